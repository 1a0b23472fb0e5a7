"""Serving operators on the GPU against their float64 oracle (``oracle.serving_oracle``)."""
import numpy as np
import pytest
import torch

from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def V():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from dsalt_b200 import serving
    return serving


def dev(x, dtype=None):
    t = torch.as_tensor(np.ascontiguousarray(x))
    return (t if dtype is None else t.to(dtype)).to("cuda", copy=True)


def status():
    from dsalt_b200 import ops
    return ops.device_status()


# ------------------------------------------------------------------ slots
@pytest.mark.parametrize("S,page,max_pages,longest,new,room,pool", [
    (1, 16, 4, 0, 1, 1, 1.0), (3, 16, 3, 40, 20, 70, 1.0), (64, 64, 20, 1200, 1, 64, 0.5), (65, 32, 9, 200, 90, 9000, 0.6),
    (1025, 128, 5, 500, 5, 5125, 0.7), (2100, 16, 6, 60, 30, 60000, 0.8), (8192, 64, 3, 120, 2, 16384, 0.9),
    (2, 64, 700, 0, 40000, 80001, 1.0)])
def test_reserve_and_release_match_the_oracle(V, S, page, max_pages, longest, new, room, pool):
    g = np.random.default_rng(S + page)
    lens = g.integers(0, longest + 1, S).astype(np.int32)
    add = g.integers(0, new + 1, S).astype(np.int32)
    add[0] = new
    held = -(-lens // page)
    wanted = int((-(-(lens + add) // page) - held).sum())
    n_free = max(1, int(wanted * pool))
    n_pages = int(held.sum()) + n_free
    ids = g.permutation(n_pages).astype(np.int32)
    tables = np.full((S, max_pages), -1, np.int32)
    at = 0
    for s in range(S):
        tables[s, :held[s]] = ids[at:at + held[s]]
        at += held[s]
    free = np.concatenate([ids[at:], np.full(at, -7, np.int32)])  # a stack with room for every page
    ref = O.reserve(tables, lens, add, free, n_free, page, room)
    for inplace in (False, True):
        t, l, f, n = dev(tables), dev(lens), dev(free), dev(np.array([n_free], np.int32))
        p = V.reserve_slots(t, l, dev(add), f, n, page, room, inplace=inplace)
        got = (t, p.slots, p.positions, p.cu_new, p.granted, p.seq_lens, p.n_free)
        for a, b, name in zip(got, ref, ("tables", "slots", "positions", "cu_new", "granted", "seq_lens", "n_free")):
            np.testing.assert_array_equal(a.cpu().numpy().reshape(np.shape(b)), b, err_msg=name)
        if inplace:
            assert p.seq_lens is l and p.n_free is n
        else:
            np.testing.assert_array_equal(l.cpu().numpy(), lens)
            assert int(n) == n_free
            l.copy_(p.seq_lens)
            n.copy_(p.n_free)
        np.testing.assert_array_equal(f.cpu().numpy(), free)
    flags = g.random(S) < 0.6
    rt, rl, rf, rn = O.release(ref[0], ref[5], flags, free, ref[6], page)
    V.release_slots(t, l, dev(flags), f, n, page)
    np.testing.assert_array_equal(t.cpu().numpy(), rt)
    np.testing.assert_array_equal(l.cpu().numpy(), rl)
    assert int(n) == rn
    np.testing.assert_array_equal(f.cpu().numpy()[:rn], rf[:rn])


def test_reserve_odd_lengths_and_states(V):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    # negative numbers count as 0; a length beyond the table is refused without being followed
    t = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    t[3, 0] = 5
    p = V.reserve_slots(t, i32(-3, 0, 1000, 4), i32(2, -5, 1, 1), i32(8, 9), i32(2), 16, 6)
    assert p.granted.tolist() == [True, True, False, True]
    assert p.seq_lens.tolist() == [2, 0, 1000, 5] and p.cu_new.tolist() == [0, 2, 2, 3, 4]
    assert p.slots.tolist() == [9 * 16, 9 * 16 + 1, -1, 5 * 16 + 4, -1, -1] and int(p.n_free) == 1
    # more free pages than the stack has entries; no room for a single token; nothing new
    t = torch.full((1, 3), -1, dtype=torch.int32, device="cuda")
    p = V.reserve_slots(t, i32(0), i32(40), i32(3, 4), i32(99), 16, 40)
    assert p.granted.tolist() == [False] and p.n_free.tolist() == [2]
    p = V.reserve_slots(t, i32(0), i32(1), i32(3, 4), i32(2), 16, 0)
    assert p.granted.tolist() == [False] and p.slots.numel() == 0 and p.cu_new.tolist() == [0, 0]
    p = V.reserve_slots(t, i32(0), i32(0), i32(3, 4), i32(0), 16, 3)
    assert p.granted.tolist() == [True] and p.slots.tolist() == [-1] * 3
    # a sum of new tokens beyond 2^31
    big = torch.full((2000,), 2**31 - 1, dtype=torch.int32, device="cuda")
    t = torch.full((2000, 1), -1, dtype=torch.int32, device="cuda")
    p = V.reserve_slots(t, torch.zeros_like(big), big, i32(1), i32(1), 16, 5)
    assert not p.granted.any() and p.slots.tolist() == [-1] * 5 and p.cu_new[-1] == 5


def test_released_pages_come_back_in_order(V):
    t = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    new = torch.tensor([40, 1, 20], dtype=torch.int32, device="cuda")
    free = torch.randperm(9, device="cuda").to(torch.int32)
    n = torch.tensor([9], dtype=torch.int32, device="cuda")
    before = free.clone()
    a = V.reserve_slots(t, lens, new, free, n, 16, 61, inplace=True)
    table = t.clone()
    V.release_slots(t, lens, torch.ones(3, dtype=torch.bool, device="cuda"), free, n, 16)
    assert (t == -1).all() and (lens == 0).all() and int(n) == 9 and torch.equal(free, before)
    b = V.reserve_slots(t, lens, new, free, n, 16, 61, inplace=True)
    assert torch.equal(a.slots, b.slots) and torch.equal(t, table)


# ------------------------------------------------------------------ append
def random_cache(g, n_pages, H, page, D, lo=-9, hi=-3):
    vals = O.VALUES[g.integers(0, 127, (n_pages, H, page, D))] * g.choice([-1.0, 1.0], (n_pages, H, page, D))
    return vals, 2.0 ** g.integers(lo, hi, (n_pages, H))


def as_f8(vals):
    return torch.from_numpy(np.ascontiguousarray(vals)).float().to(F8).cuda()


def check_append(V, k, v, cache, slots, page, k_dev=None, v_dev=None):
    (kc, ks), (vc, vs) = cache
    dk, dv, dks, dvs = as_f8(kc), as_f8(vc), dev(ks, torch.float32), dev(vs, torch.float32)
    V.append_cache(k.cuda() if k_dev is None else k_dev, v.cuda() if v_dev is None else v_dev, dk, dv, dks, dvs, dev(slots))
    for x, (c, s), gc, gs in ((k, cache[0], dk, dks), (v, cache[1], dv, dvs)):
        rc, rs = O.append(x.double().numpy(), c, s, slots, page)
        np.testing.assert_array_equal(gs.cpu().double().numpy(), rs)
        np.testing.assert_array_equal(gc.double().cpu().numpy(), rc)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,D,page,runs", [
    (1, 64, 16, [(3, 0, 1)]), (2, 128, 16, [(0, 5, 11), (1, 0, 16), (2, 0, 16), (4, 0, 3)]),
    (3, 64, 64, [(7, 63, 1), (6, 0, 64), (5, 10, 40)]), (2, 128, 128, [(1, 0, 128), (0, 100, 28), (2, 127, 1)]),
    (16, 64, 64, [(i, (5 * i) % 64, 1) for i in range(9)]), (1, 128, 32, [(i, 0, 32) for i in range(40)]),
    (5, 64, 32, [(i, 3 * i % 30, 2) for i in range(70)])])
def test_append_matches_the_oracle(V, dtype, H, D, page, runs):
    g = np.random.default_rng(len(runs) * D + page)
    slots = np.concatenate([np.arange(n) + p * page + off for p, off, n in runs]).astype(np.int64)
    n_pages = max(p for p, _, _ in runs) + 2
    T = len(slots)
    tg = torch.Generator().manual_seed(T)
    k = (torch.randn(T, H, D, generator=tg) * 2.0 ** torch.randint(-6, 5, (T, 1, 1), generator=tg)).to(dtype)
    v = torch.randn(T, H, D, generator=tg).to(dtype)
    cache = random_cache(g, n_pages, H, page, D), random_cache(g, n_pages, H, page, D, -14, 3)
    check_append(V, k, v, cache, slots, page)


def test_append_strided_rows_and_skipped_slots(V):
    g = np.random.default_rng(5)
    H, D, page, T = 3, 64, 16, 37
    qkv = torch.randn(T, 3 * H, D + 8, generator=torch.Generator().manual_seed(1)).bfloat16()
    slots = np.arange(T, dtype=np.int64) + 20
    slots[[0, 7, 30, 31, 36]] = [-1, -5, 10 ** 9, -1, 6 * 16]  # none, none, beyond the pool, none, beyond the pool
    cache = random_cache(g, 6, H, page, D), random_cache(g, 6, H, page, D)
    qd = qkv.cuda()
    k, v = qkv[:, H:2 * H, :D], qkv[:, 2 * H:, 8:]
    # heads D + 8 apart, 16-byte aligned: taken as they are; an odd offset: copied first
    check_append(V, k, v, cache, slots, page, qd[:, H:2 * H, :D], qd[:, 2 * H:, 8:])
    k, v = qkv[:, H:2 * H, 1:D + 1], qkv[:, 2 * H:, 3:D + 3]
    check_append(V, k, v, cache, slots, page, qd[:, H:2 * H, 1:D + 1], qd[:, 2 * H:, 3:D + 3])
    # nothing to write
    check_append(V, k, v, cache, np.full(T, -1, np.int64), page)
    check_append(V, k[:0], v[:0], cache, np.zeros(0, np.int64), page)


def test_append_extreme_values(V):
    g = np.random.default_rng(6)
    H, D, page = 1, 64, 16
    rows = torch.zeros(10, H, D)
    rows[1] = 3.0e38
    rows[2] = 1e-38          # below the smallest scale
    rows[3] = 1e-44          # a denormal
    rows[4, 0, :5] = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0, -1.75])
    rows[5] = float("nan")
    rows[6] = float("inf")
    rows[7, 0, :3] = torch.tensor([448.0, 448.1, -447.0])
    rows[8, 0, :3] = torch.tensor([1.75, 2.0 ** -17, 1.75 * 2.0 ** -18])  # subnormal bytes and their ties
    rows[9] = -0.0
    cache = random_cache(g, 10, H, page, D), random_cache(g, 10, H, page, D, -100, -60)
    cache[0][1][2] = 0.0  # scales of pages never written
    cache[0][1][5] = 0.0
    for off in (0, 3):    # afresh; onto older tokens (values that sink to nothing among them)
        slots = np.arange(10, dtype=np.int64) * page + off
        check_append(V, rows, rows.flip(0), cache, slots, page)


def test_append_token_by_token_equals_the_oracle_and_keeps_other_pages(V):
    g = np.random.default_rng(7)
    H, D, page, n = 2, 64, 16, 48
    x = (torch.randn(n, H, D, generator=torch.Generator().manual_seed(3)) *
         torch.logspace(-2, 2, n)[:, None, None]).bfloat16()  # the scale grows again and again
    ref = cache = random_cache(g, 5, H, page, D)
    dk, ds = as_f8(cache[0]), dev(cache[1], torch.float32)
    dv, dvs = dk.clone(), ds.clone()
    order = [3, 0, 4]
    slots = np.concatenate([np.arange(page) + p * page for p in order])
    for t in range(n):
        V.append_cache(x[t:t + 1].cuda(), x[t:t + 1].cuda(), dk, dv, ds, dvs, dev(slots[t:t + 1]))
        ref = O.append(x[t:t + 1].double().numpy(), *ref, slots[t:t + 1], page)
    np.testing.assert_array_equal(dk.double().cpu().numpy(), ref[0])
    np.testing.assert_array_equal(ds.cpu().numpy(), ref[1])
    assert torch.equal(dk.view(torch.uint8), dv.view(torch.uint8)) and torch.equal(ds, dvs)
    np.testing.assert_array_equal(dk.double().cpu().numpy()[[1, 2]], cache[0][[1, 2]])


# ------------------------------------------------------------------ attention
def attend_case(seed, lens, q_lens, H, Hkv, D, page, dtype, w_max=0, k_lmk=0, bias=False, e=((-9, -4), (-9, -4)), q_size=1.0):
    g = np.random.default_rng(seed)
    S, T = len(lens), int(sum(q_lens))
    pages = [-(-n // page) for n in lens]
    n_pages = sum(pages) + 2
    ids = g.permutation(n_pages)
    max_pages = max(max(pages), 1) + 1
    tables = np.full((S, max_pages), -1, np.int32)
    at = 0
    for s in range(S):
        tables[s, :pages[s]] = ids[at:at + pages[s]]
        at += pages[s]
    kc, ks = random_cache(g, n_pages, Hkv, page, D, *e[0])
    vc, vs = random_cache(g, n_pages, Hkv, page, D, *e[1])
    q = (torch.from_numpy(g.normal(size=(T, H, D))).float() * q_size).to(dtype)
    w = lmk = b = None
    if w_max:
        w = g.integers(1, w_max + 1, T).astype(np.int32)
        if k_lmk:
            lmk = np.full((H, S, k_lmk), -1, np.int32)
            for h in range(H):
                for s in range(S):
                    m = min(int(g.integers(0, k_lmk + 1)), lens[s])
                    lmk[h, s, :m] = g.permutation(lens[s])[:m]  # any order
                    lmk[h, s] = g.permutation(lmk[h, s])
            if bias:
                b = g.normal(size=lmk.shape).astype(np.float32)
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    return dict(q=q, kc=kc, vc=vc, ks=ks, vs=vs, tables=tables, lens=np.array(lens, np.int32), cu=cu, w=w, lmk=lmk, bias=b)


def to_gpu(c):
    o = lambda x, dt=None: None if x is None else dev(x, dt)  # noqa: E731
    return dict(q=c["q"].cuda(), k_cache=as_f8(c["kc"]), v_cache=as_f8(c["vc"]), k_scale=dev(c["ks"], torch.float32),
                v_scale=dev(c["vs"], torch.float32), block_tables=dev(c["tables"]), seq_lens=dev(c["lens"]),
                cu_q=o(c["cu"]), w_sizes=o(c["w"]), lmk_indices=o(c["lmk"]), lmk_bias=o(c["bias"]))


def oracle_of(c):
    return O.attention(c["q"].double().numpy(), c["kc"], c["vc"], c["ks"], c["vs"], c["tables"], c["lens"], c["cu"], c["w"],
                       c["lmk"], None if c["bias"] is None else c["bias"].astype(np.float64))


def check_attend(c, out, lse, what=""):
    """Bound of a row's error, before the result's own rounding (half a step of its type):
    * logits: an fp32 sum of D exact products and a few operations, each within 2^-22 of the sum of
      magnitudes (tensor-core accumulation may drop bits instead of rounding): E = (D + 8) 2^-22 size,
      plus |x| 2^-22 for the change of base and 2 ulp of exp2; p is off by a factor exp(E)
    * P: half a step of fp16, 2^-11, per element; with two terms 2^-22
    * sums of n terms in fp32: (n + 8) 2^-22, an upper bound whatever their order
    out = sum p v / sum p, so each of these counts at most twice, relative to sum p|v| / sum p."""
    ref, rl, spread, size, n = oracle_of(c)
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    D = ref.shape[2]
    fp32 = c["q"].dtype == torch.float32
    half = torch.finfo(c["q"].dtype).eps / 2
    # below the smallest normal number 2^-14 fp16 has a fixed step of 2^-24: half a step is 2^-25 whatever
    # the value (bf16 and fp32 likewise, at 2^-134 and 2^-150)
    flat = torch.finfo(c["q"].dtype).smallest_normal * half
    live = np.isfinite(rl)
    E = np.where(live, (D + 8) * 2.0 ** -22 * size + (np.abs(np.where(live, rl, 0)) + 1) * 2.0 ** -21, 0)
    E = E + (n + 8) * 2.0 ** -22
    tol = half * np.abs(ref) * (1 + 2 ** -8) + (2 * np.expm1(E) + (2.0 ** -21 if fp32 else 2.0 ** -11))[..., None] * spread
    assert (out[~live] == 0).all() and np.isneginf(lse[~live]).all(), what
    err = np.abs(out - ref)
    bad = ~(err <= tol + flat + 1e-30)
    assert not bad.any(), f"{what}: {bad.sum()} values, worst {np.nanmax(err / (tol + flat + 1e-30)):.3f} of the bound"
    lse_err = np.abs(np.where(live, lse - np.where(live, rl, 0), 0))
    assert (lse_err <= E + 2.0 ** -22 * (np.abs(np.where(live, rl, 0)) + 1)).all(), what


def run_attend(V, c, **kw):
    out, lse = V.cache_attention(**{**to_gpu(c), **kw}, return_lse=True)
    check_attend(c, out, lse)
    assert status() == 0
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D,page,lens,q_lens", [
    (1, 1, 64, 16, [1], [1]), (4, 4, 64, 16, [1, 15, 16, 17, 0, 33], [1] * 6), (16, 2, 128, 64, [257, 63, 64, 65], [1] * 4),
    (6, 2, 64, 32, [100, 5, 40], [3, 5, 0]), (5, 1, 128, 128, [300, 129], [7, 1]), (20, 1, 64, 16, [50, 90], [1, 4]),
    (40, 2, 128, 32, [70], [2]), (8, 8, 64, 64, [2, 700], [4, 2])])
def test_attention_over_every_key(V, dtype, H, Hkv, D, page, lens, q_lens):
    run_attend(V, attend_case(1, lens, q_lens, H, Hkv, D, page, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,Hkv,D,page,lens,q_lens,w_max,k,bias", [
    (4, 4, 64, 16, [1, 2, 100, 300, 17], [1] * 5, 40, 12, False), (16, 2, 128, 64, [400, 64, 3], [1] * 3, 100, 33, True),
    (6, 2, 64, 32, [90, 200, 1], [5, 2, 1], 60, 16, True), (12, 12, 64, 64, [500], [1], 512, 64, False),
    (5, 1, 128, 128, [260, 130], [3, 7], 1, 17, True), (20, 2, 64, 16, [150, 33], [2, 3], 30, 5, False),
    (4, 2, 64, 64, [70, 5], [1, 1], 30, 0, False), (2, 2, 128, 16, [600], [8], 500, 128, True)])
def test_attention_over_windows_and_landmarks(V, dtype, H, Hkv, D, page, lens, q_lens, w_max, k, bias):
    run_attend(V, attend_case(2, lens, q_lens, H, Hkv, D, page, dtype, w_max, k, bias))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[2500], [1500, 7, 900], [300] * 40, [3] * 127 + [400], [3] * 128 + [0, 900], [1, 60] * 700])
def test_attention_with_cut_keys(V, D, lens):
    # keys split over blocks, short sequences beside long ones
    run_attend(V, attend_case(3, lens, [1] * len(lens), 2, 1, D, 64, torch.bfloat16))


@pytest.mark.parametrize("H,Hkv,D,page,lens,q_lens,w_max,k", [
    (4, 2, 64, 16, [420, 900], [300, 2], 90, 40), (8, 1, 128, 64, [261, 0, 40], [261, 0, 35], 70, 33),
    (2, 2, 64, 32, [700], [513], 0, 0), (3, 1, 64, 16, [30] * 9, [30] * 9, 12, 5), (2, 1, 64, 16, [20, 3, 50], [40, 9, 12], 30, 8),
    (16, 2, 64, 64, [600, 8], [8, 8], 2**31 - 1, 20), (3, 1, 64, 16, [500, 77, 9], [9, 15, 3], 100, 64)])
def test_attention_of_many_tokens_per_sequence(V, H, Hkv, D, page, lens, q_lens, w_max, k):
    run_attend(V, attend_case(5, lens, q_lens, H, Hkv, D, page, torch.bfloat16, w_max, k))


def test_single_tokens_and_heads_of_any_stride(V):
    # a dimension of one element may have any stride, an expanded row the stride 0
    c = attend_case(6, [40], [1], 1, 1, 64, 16, torch.bfloat16)
    plain, args = to_gpu(c)["q"], to_gpu(c)
    for strides in ((1, 1, 1), (0, 0, 1), (7, 3, 1)):
        args["q"] = plain.as_strided((1, 1, 64), strides)
        out, lse = V.cache_attention(**args, return_lse=True)
        check_attend(c, out, lse)
    c = attend_case(7, [40, 33], [1, 1], 2, 1, 64, 16, torch.bfloat16)
    args = to_gpu(c)
    args["q"] = args["q"][:1].expand(2, -1, -1)
    same = dict(args, q=args["q"].contiguous())
    assert torch.equal(V.cache_attention(**args), V.cache_attention(**same))
    k = torch.randn(64, device="cuda").to(torch.bfloat16)
    caches = [[torch.zeros(2, 1, 16, 64, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
              + [torch.zeros(2, 1, device="cuda") for _ in range(2)] for _ in range(2)]
    slot = torch.tensor([17], device="cuda")
    V.append_cache(k.as_strided((1, 1, 64), (1, 5, 1)), k.as_strided((1, 1, 64), (0, 0, 1)), *caches[0], slot)
    V.append_cache(k.view(1, 1, 64), k.view(1, 1, 64), *caches[1], slot)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_long_uncut_rows_loses_nothing_on_the_way(V, D, dtype):
    # More sequences than places, so that none is cut: each warp adds up 65536 keys of positive V.
    # What a rounding or a cut of the running sum may cost, relative to the result:
    # * fp16 P: half a step of 2^-11 per key, either sign: 8 * 2^-11 / sqrt(131072) = 1.1e-5;
    # * at most 128 products in a row, each cut by one step of 2^-23 of a sum that grows evenly:
    #   64 * 2^-23 = 7.6e-6;
    # * fp32 sums with rounding, at most 4096 of them, either sign, growing evenly:
    #   8 * 2^-24 * sqrt(4096 / 3) = 1.8e-5 (fp32 queries; 32 of them, 1.6e-6, for the others).
    # Both kinds stay below 3e-5; 4096 products in a row, each cut, come to 2e-4 and more.
    S, n, page = 1200, 131072, 128
    g = torch.Generator(device="cuda").manual_seed(D)
    k = torch.randn(n // page, 1, page, D, device="cuda", generator=g).to(F8)
    v = (torch.rand(n // page, 1, page, D, device="cuda", generator=g) + 0.5).to(F8)
    scale = torch.ones(n // page, 1, device="cuda")
    tables = torch.arange(n // page, device="cuda", dtype=torch.int32).repeat(S, 1)
    q = (torch.randn(S, 1, D, device="cuda", generator=g) * 0.3).to(dtype)
    out = V.cache_attention(q, k, v, scale, scale, tables, torch.full((S,), n, device="cuda", dtype=torch.int32),
                            out_dtype=torch.float32)
    some = torch.arange(0, S, 97, device="cuda")
    x = q[some, 0].double() @ k.double().reshape(n, D).T / D ** 0.5
    want = torch.softmax(x, -1) @ v.double().reshape(n, D)
    assert ((out[some, 0].double() - want) / want).abs().max().item() < 3e-5


def test_attention_widths_and_landmarks_at_their_limits(V):
    c = attend_case(4, [200, 90, 64], [2, 1, 1], 4, 2, 64, 16, torch.float16, 50, 9, True)
    c["w"] = np.array([0, -7, 2**31 - 1, 90], np.int32)  # below 1: 1; beyond the start: every key
    c["lmk"][0, 0] = [198, 199, 200, 10**9, -1, -2**31, 0, 197, 3]  # own position, behind it, far off, none
    run_attend(V, c)
    c["bias"][:] = -np.inf  # a landmark without weight
    run_attend(V, c)
    c["bias"][:] = 0
    c["bias"][1, 0, :3] = 60.0  # landmarks that take everything
    run_attend(V, c)


def test_attention_scales_far_apart(V):
    # pages whose scales lie 2^200 apart, pages of zeros and pages never written (scale 0)
    for seed, e in ((5, ((-9, -4), (-110, 110))), (6, ((-40, -3), (-9, -4)))):
        c = attend_case(seed, [700, 130], [1, 3], 4, 2, 64, 16, torch.bfloat16, e=e)
        run_attend(V, c)
    c = attend_case(7, [640], [1], 2, 2, 64, 16, torch.bfloat16, e=((-9, -4), (0, 20)))
    p = c["tables"][0, ::2][:20]
    c["vc"][p], c["vs"][p] = 0.0, 2.0 ** -110
    run_attend(V, c)
    c["ks"][p], c["vs"][p] = 0.0, 0.0
    run_attend(V, c)


def test_attention_query_sizes(V):
    for size in (2.0 ** -100, 2.0 ** 60):
        c = attend_case(8, [90, 40], [1, 2], 4, 2, 64, 16, torch.bfloat16, e=((-9, -4), (-9, -4)), q_size=size)
        c["ks"] = c["ks"] / size if size > 1 else c["ks"]
        run_attend(V, c)
    c = attend_case(8, [90], [1], 2, 2, 64, 16, torch.float32)
    c["q"][0, 1] = 0.0
    c["q"][0, 0, 0] = 1e30  # one element that hides the others
    c["kc"][:, 0, :, 0] = 0.0
    c["ks"][:] = 2.0 ** -9
    out, lse = V.cache_attention(**to_gpu(c), return_lse=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_attention_nan_stays_with_the_keys_that_hold_it(V):
    c = attend_case(9, [150, 90], [3, 1], 4, 2, 64, 16, torch.bfloat16, 30, 7)
    c["w"] = np.array([20, 9, 30, 12], np.int32)
    base, _ = run_attend(V, c)
    gpu = to_gpu(c)
    page = 16

    def poison(s, pos, hk, name, where):
        x = gpu[name].view(torch.uint8)
        x[int(c["tables"][s, pos // page]), hk, pos % page, where] = 0x7f

    # a value of key 139 of kv head 0: of the queries at 147, 148, 149 only those whose window (or
    # landmark list) holds it may see it, in that channel alone
    poison(0, 139, 0, "v_cache", 5)
    poison(0, 140, 1, "k_cache", 6)   # a key's channel: every channel of the queries that see it
    poison(1, 3, 0, "v_cache", 0)
    out, lse = V.cache_attention(**gpu, return_lse=True)
    want_v, want_k = np.zeros((4, 4), bool), np.zeros((4, 4), bool)
    for t, (s, i) in enumerate([(0, 147), (0, 148), (0, 149), (1, 89)]):
        lo = max(0, i - int(c["w"][t]) + 1)
        sees = lambda h, p: lo <= p <= i or (p < lo and p in c["lmk"][h, s])  # noqa: E731
        for h in range(4):
            want_v[t, h] = sees(h, 139) if s == 0 and h < 2 else (s == 1 and h < 2 and sees(h, 3))
            want_k[t, h] = s == 0 and h >= 2 and sees(h, 140)
    assert want_v.any() and want_k.any() and not want_v.all()
    nan = torch.isnan(out).cpu().numpy()
    for t in range(4):
        for h in range(4):
            expect = np.zeros(64, bool)
            expect[5 if t < 3 else 0] = want_v[t, h]
            expect |= want_k[t, h]
            np.testing.assert_array_equal(nan[t, h], expect, err_msg=f"{t} {h}")
    clean = ~nan & ~want_k[..., None]
    assert torch.equal(out.cpu()[torch.from_numpy(clean)], base.cpu()[torch.from_numpy(clean)])
    assert status() == 0


def test_attention_bytes_behind_the_end_do_not_count(V):
    c = attend_case(10, [37, 130, 1], [1, 2, 1], 4, 2, 128, 64, torch.float16, 20, 5)
    base, lse0 = run_attend(V, c)
    gpu = to_gpu(c)
    for s, n in enumerate(c["lens"]):
        last = int(c["tables"][s, (n - 1) // 64])
        for name in ("k_cache", "v_cache"):
            gpu[name].view(torch.uint8)[last, :, n % 64 if n % 64 else 64:] = 0x7f  # NaN
    out, lse = V.cache_attention(**gpu, return_lse=True)
    assert torch.equal(out, base) and torch.equal(lse, lse0)


def test_attention_rows_behind_the_last_sequence_and_empty_ones(V):
    for D in (64, 128):
        rows_behind(V, attend_case(11, [50, 0, 9], [2, 1, 1], 4, 2, D, 16, torch.bfloat16))
    # more query tokens than the sequence has: those before its start have no keys
    c = attend_case(12, [2, 60], [4, 1], 4, 2, 64, 16, torch.bfloat16)
    out, _ = run_attend(V, c)
    assert (out[:2] == 0).all()
    # no rows at all
    gpu = to_gpu(c)
    gpu["cu_q"] = torch.zeros(3, dtype=torch.int32, device="cuda")
    out = V.cache_attention(**{**gpu, "q": gpu["q"][:0]})
    assert out.shape == (0, 4, 64)
    out = V.cache_attention(**gpu)
    assert (out == 0).all()


def rows_behind(V, c):
    gpu = to_gpu(c)
    gpu["q"] = torch.cat([gpu["q"], torch.full((5, *c["q"].shape[1:]), float("nan"), dtype=torch.bfloat16, device="cuda")])
    out, lse = V.cache_attention(**gpu, return_lse=True)
    check_attend(c, out[:4], lse[:4])
    assert (out[4:] == 0).all() and torch.isneginf(lse[4:]).all()
    assert (out[2] == 0).all()  # a query of an empty sequence


def test_attention_bad_pages_are_left_out_and_reported(V):
    from dsalt_b200 import ops
    c = attend_case(13, [100, 40], [1, 1], 2, 1, 64, 16, torch.bfloat16)
    c["tables"][0, 2] = 10**8
    c["tables"][0, 4] = -1
    c["tables"][1, 0] = -2**31
    out, lse = V.cache_attention(**to_gpu(c), return_lse=True)
    check_attend(c, out, lse)
    assert ops.device_status() != 0 and ops.device_status() == 0
    c["lens"][1] = 10**9  # a length beyond the table: the table's end counts
    out = V.cache_attention(**to_gpu(c))
    assert torch.equal(out[0], V.cache_attention(**to_gpu(c))[0])
    ops.device_status()


def test_attention_strided_queries_types_and_refusals(V):
    c = attend_case(14, [80, 33], [1, 1], 4, 2, 64, 16, torch.bfloat16, 20, 4)
    gpu = to_gpu(c)
    qkv = torch.zeros(2, 8 * 64 + 8, dtype=torch.bfloat16, device="cuda")
    for off in (0, 8, 3):  # in place; copied for its odd offset
        q = qkv[:, off:off + 4 * 64].view(2, 4, 64)
        q.copy_(gpu["q"])
        out, lse = V.cache_attention(**{**gpu, "q": q}, return_lse=True)
        check_attend(c, out, lse)
    out32 = V.cache_attention(**gpu, out_dtype=torch.float32)
    assert out32.dtype == torch.float32 and torch.equal(out32.bfloat16(), V.cache_attention(**gpu))
    for change, err in ((dict(w_sizes=None), ValueError), (dict(seq_lens=gpu["seq_lens"].long()), TypeError),
                        (dict(q=gpu["q"][:, :3]), ValueError), (dict(cu_q=gpu["cu_q"][:2]), ValueError),
                        (dict(lmk_indices=gpu["lmk_indices"][:, :1]), ValueError), (dict(cu_q=None, q=gpu["q"][:1]), ValueError),
                        (dict(k_cache=gpu["k_cache"].view(torch.uint8)), TypeError), (dict(q=gpu["q"].double()), TypeError),
                        (dict(block_tables=gpu["block_tables"].t()), ValueError),
                        (dict(lmk_indices=None, lmk_bias=gpu["k_scale"]), ValueError)):
        with pytest.raises(err):
            V.cache_attention(**{**gpu, **change})


def test_attention_is_deterministic_and_follows_a_captured_graph(V):
    c = attend_case(15, [1200, 90, 400], [1, 1, 1], 4, 2, 64, 64, torch.bfloat16, 300, 20)
    c["cu"] = None
    full = dict(to_gpu(c), w_sizes=None, lmk_indices=None)
    both = [to_gpu(c), full]
    torch.cuda.synchronize()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for g in both:
        V.cache_attention(**g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(V.cache_attention(**g, return_lse=True))
        graphs.append(graph)
    for lens in ([1200, 90, 400], [3, 0, 399], [1100, 64, 16]):
        for g in both:
            g["seq_lens"].copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        graphs[0].replay()            # two graphs at once, on two streams
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for g, (o, l) in zip(both, outs):
            eo, el = V.cache_attention(**g, return_lse=True)
            assert torch.equal(o, eo) and torch.equal(l, el)
            d = dict(c, lens=np.array(lens, np.int32))
            check_attend(d if g is both[0] else dict(d, w=None, lmk=None), o, l)
    assert status() == 0


# ------------------------------------------------------------------ sampling
def check_sample(V, logits, u, t=1.0, k=0, p=1.0, m=0.0):
    tok, lp = V.sample_tokens(logits, u, temperature=t, top_k=k, top_p=p, min_p=m, return_logprob=True)
    tok, lp = tok.cpu().numpy(), lp.cpu().numpy()
    row = lambda v, i: float(v[i]) if isinstance(v, torch.Tensor) else float(np.float32(v))  # noqa: E731
    l, un = logits.double().cpu().numpy(), u.double().cpu().numpy()
    skipped = 0
    for i in range(len(l)):
        rt, rl, margin = O.sample(l[i], un[i], row(t, i), int(row(k, i)), row(p, i), row(m, i))
        # a prefix and the total are each off by at most V roundings of 2^-44, and the total is at least 1
        if margin < 2.0 ** -43 * l.shape[1]:
            skipped += 1
            continue
        assert tok[i] == rt, (i, tok[i], rt, margin)
        assert lp[i] == rl or abs(lp[i] - rl) <= 2.0 ** -23 * (abs(rl) + 1), (i, lp[i], rl)
    assert skipped <= 0.1 * len(l) + 1


FILTERS = {"none": {}, "greedy": dict(t=0.0), "k1": dict(k=1), "k50": dict(t=0.8, k=50), "k5000": dict(t=1.5, k=5000),
           "p": dict(t=1.0, p=0.9), "p_flat": dict(t=30.0, p=0.7), "m": dict(m=0.05), "p0": dict(p=0.0),
           "all": dict(t=0.8, k=50, p=0.9, m=0.02), "k_p_wide": dict(t=20.0, k=3000, p=0.8), "cold": dict(t=1e-30, p=0.5),
           "m1": dict(t=2.0, m=1.0)}


@pytest.mark.parametrize("name", list(FILTERS))
@pytest.mark.parametrize("B,Vn,dtype", [(3, 1, torch.float32), (5, 33, torch.float16), (2, 1000, torch.bfloat16),
                                        (4, 50257, torch.float32), (40, 50257, torch.bfloat16), (2, 151936, torch.float16)])
def test_sample_matches_the_oracle(V, name, B, Vn, dtype):
    g = torch.Generator(device="cuda").manual_seed(B + Vn)
    logits = (torch.randn(B, Vn, device="cuda", generator=g) * 2.5).to(dtype)
    check_sample(V, logits, torch.rand(B, device="cuda", generator=g), **FILTERS[name])


@pytest.mark.parametrize("name", ["none", "k50", "k5000", "p", "all", "m1"])
def test_sample_equal_logits(V, name):
    # every logit equal; and two values only: the order of equal logits is their index
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.tensor([0.0, 0.25, 0.999, 0.61], device="cuda")
    flat = torch.full((4, 20000), -3.25, device="cuda", dtype=torch.bfloat16)
    two = torch.where(torch.rand(4, 20000, device="cuda", generator=g) < 0.4, 1.0, 0.5).half()
    check_sample(V, two, torch.rand(4, device="cuda", generator=g), **FILTERS[name])
    if name not in ("p", "all"):  # p * V may hit a border exactly
        check_sample(V, flat, u + 1e-5 * (u < 0.9), **FILTERS[name])
    tok = V.sample_tokens(flat, u, top_k=7, top_p=0.5)
    assert tok.tolist() == [0, 1, 3, 2]  # 4 of 7 kept


def test_sample_masked_and_odd_logits(V):
    inf, nan = float("inf"), float("nan")
    rows = torch.tensor([[-inf, 1.0, nan, 2.0, -inf], [-inf, -inf, -inf, -inf, -inf], [nan, nan, nan, nan, nan],
                         [inf, 0.0, inf, 1.0, -inf], [-3.4e38, -inf, -3.4e38, -inf, nan], [0.0, -0.0, 0.0, -0.0, 0.0],
                         [3.4e38, -3.4e38, 3.4e38, 0.0, 1.0]], device="cuda")
    for u in (0.0, 0.3, 0.7, 0.9999):
        uu = torch.full((7,), u, device="cuda")
        for f in ({}, dict(k=2), dict(p=0.6), dict(t=0.0), dict(t=0.5, m=0.3), dict(t=3e38)):
            if u == 0.0 and f.get("p"):
                continue
            check_sample(V, rows, uu + 0.013, **f)
    # the lowest finite number as the largest logit; temperatures at which one step of fp32 is everything
    low = -torch.finfo(torch.float32).max
    edge = torch.tensor([[-inf, low, -inf, low, low], [0.0, -1e-45, 0.0, 1e-45, -inf], [1.0, 1.0 - 2**-24, 1.0, -1.0, 0.5]],
                        device="cuda")
    for t in (1e-45, 1e-38, 1e-30, 1e-3, 1.0, 3e38):
        for f in ({}, dict(p=0.4), dict(k=2)):
            check_sample(V, edge, torch.full((3,), 0.57, device="cuda"), t=t, **f)
    tok, lp = V.sample_tokens(rows, torch.full((7,), 0.9, device="cuda"), return_logprob=True)
    assert tok.tolist()[1:4] == [0, 0, 2] and lp[1] == -inf and lp[2] == -inf
    # uniforms outside [0, 1): the nearest token
    lg = torch.zeros(4, 9, device="cuda")
    assert V.sample_tokens(lg, torch.tensor([-1.0, 1.0, 5.0, nan], device="cuda")).tolist() == [0, 8, 8, 0]
    # large masked rows: what is left lies anywhere
    big = torch.full((3, 50257), -inf, device="cuda", dtype=torch.bfloat16)
    big[0, 50256] = 0
    big[1, 17], big[1, 40000] = -200.0, -200.0
    big[2, 5000:5010] = torch.arange(10, device="cuda").bfloat16()
    for f in ({}, dict(k=3), dict(p=0.5), dict(k=2000, p=0.99)):
        check_sample(V, big, torch.tensor([0.5, 0.75, 0.4], device="cuda"), **f)


def test_sample_per_row_settings_strides_and_batch_independence(V):
    g = torch.Generator(device="cuda").manual_seed(3)
    B, Vn = 37, 33001
    wide = (torch.randn(B, Vn + 7, device="cuda", generator=g) * 3).bfloat16()
    u = torch.rand(B, device="cuda", generator=g)
    pick = lambda v, dt: torch.tensor(v, dtype=dt, device="cuda")[torch.arange(B, device="cuda") % len(v)].contiguous()  # noqa: E731
    t, k = pick([0.0, 0.7, 1.0, 1.7, 25.0], torch.float32), pick([0, 20, -4, 1500, 10**9, 1, 2**31 - 1], torch.int32)
    p, m = pick([1.0, 0.9, 2.0, 0.3], torch.float32), pick([0.0, 0.1, -1.0], torch.float32)
    for off in (0, 1, 5):  # rows that start on any byte pair
        lg = wide[:, off:off + Vn]
        check_sample(V, lg, u, t, k, p, m)
        whole = V.sample_tokens(lg, u, temperature=t, top_k=k, top_p=p, min_p=m)
        for i in (0, 3, 17, 36):
            one = V.sample_tokens(lg[i:i + 1], u[i:i + 1], temperature=t[i:i + 1], top_k=k[i:i + 1], top_p=p[i:i + 1],
                                  min_p=m[i:i + 1])
            assert one[0] == whole[i]
        for _ in range(3):
            assert torch.equal(whole, V.sample_tokens(lg, u, temperature=t, top_k=k, top_p=p, min_p=m))
    # a transposed matrix is copied first
    tr = wide[:, :Vn].t().contiguous().t()
    assert torch.equal(V.sample_tokens(tr, u), V.sample_tokens(wide[:, :Vn], u))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_largest_vocabulary_and_batch(V, dtype):
    g = torch.Generator(device="cuda").manual_seed(4)
    lg = (torch.randn(2, 1 << 20, device="cuda", generator=g) * 2).to(dtype)  # beyond what shared memory holds
    u = torch.rand(2, device="cuda", generator=g)
    for f in ({}, dict(k=40), dict(k=4000), dict(p=0.9), dict(t=0.3, p=0.5, m=0.01)):
        check_sample(V, lg, u, **f)
    with pytest.raises(Exception, match="2\\^20"):
        V.sample_tokens(torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1])
    many = (torch.randn(1500, 700, device="cuda", generator=g) * 2).to(dtype)
    check_sample(V, many, torch.rand(1500, device="cuda", generator=g), t=0.9, k=100, p=0.95)
    assert V.sample_tokens(many[:0], u[:0]).shape == (0,)


# ------------------------------------------------------------------ graphs, streams, the operators together
def test_a_captured_decode_step_follows_the_state(V):
    """Slots, append, attention and sampling in one graph, on a stream of its own; each replay is a
    step, and equals the same calls made one by one on a copy of the state."""
    S, H, Hkv, D, page, max_pages, n_pages = 3, 4, 2, 64, 16, 6, 20
    g = torch.Generator(device="cuda").manual_seed(1)
    new = torch.tensor([1, 1, 0], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(S, Hkv, D, device="cuda", generator=g).bfloat16() for _ in range(2))
    q, head = torch.randn(S, H, D, device="cuda", generator=g).bfloat16(), torch.randn(H * D, 500, device="cuda", generator=g)
    u = torch.rand(S, device="cuda", generator=g)

    def state():
        kc = torch.zeros(n_pages, Hkv, page, D, device="cuda").to(F8)
        sc = torch.zeros(n_pages, Hkv, device="cuda")
        t = torch.full((S, max_pages), -1, dtype=torch.int32, device="cuda")
        t[0, 0], t[2, 0] = 18, 19  # the pages of the tokens already there
        return dict(t=t, n=torch.tensor([14, 0, 3], dtype=torch.int32, device="cuda"),
                    free=torch.arange(n_pages, dtype=torch.int32, device="cuda"),
                    nf=torch.tensor([18], dtype=torch.int32, device="cuda"), kc=kc, vc=kc.clone(), ks=sc, vs=sc.clone())

    def step(s):
        plan = V.reserve_slots(s["t"], s["n"], new, s["free"], s["nf"], page, S, inplace=True)
        V.append_cache(k, v, s["kc"], s["vc"], s["ks"], s["vs"], plan.slots)
        out = V.cache_attention(q, s["kc"], s["vc"], s["ks"], s["vs"], s["t"], s["n"], cu_q=plan.cu_new)
        tok, lp = V.sample_tokens(out.flatten(1).float() @ head, u, temperature=0.7, top_k=40, top_p=0.9, return_logprob=True)
        return plan.slots, plan.positions, out, tok, lp

    a, b = state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(state())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = step(a)
        for _ in range(20):
            graph.replay()
            for x, y in zip(captured, step(b)):
                assert torch.equal(x, y)
    side.synchronize()
    assert a["n"].tolist() == [34, 20, 3] and torch.equal(a["t"], b["t"]) and int(a["nf"]) == 18 - 2 - 2
    assert status() == 0


def test_offsets_beyond_32_bits(V):
    # a cache of more than 2^32 bytes a side, tokens and rows more than 2^31 elements apart
    Hkv, page, D = 2, 128, 128
    n_pages = (1 << 32) // (Hkv * page * D) + 3
    ids = [n_pages - 1, n_pages // 2 + 1, n_pages - 2, 0]
    big = [torch.empty(n_pages, Hkv, page, D, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
    big += [torch.zeros(n_pages, Hkv, device="cuda") for _ in range(2)]
    small = [torch.empty(4, Hkv, page, D, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
    small += [torch.zeros(4, Hkv, device="cuda") for _ in range(2)]
    T = 4 * page - 5
    g = torch.Generator(device="cuda").manual_seed(11)
    k, v = (torch.randn(T, Hkv, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    within = torch.arange(T, device="cuda") % page
    slots = lambda pages: torch.tensor(pages, device="cuda")[torch.arange(T, device="cuda") // page] * page + within  # noqa: E731
    V.append_cache(k, v, *big, slots(ids))
    V.append_cache(k, v, *small, slots([0, 1, 2, 3]))
    for a, b in zip(big, small):
        a = a.view(torch.uint8) if a.dtype == F8 else a
        b = b.view(torch.uint8) if b.dtype == F8 else b
        for i, p in enumerate(ids):
            n = min(page, T - i * page)
            assert torch.equal(a[p][:, :n] if a.dim() == 4 else a[p], b[i][:, :n] if b.dim() == 4 else b[i])
    q = torch.randn(1, 4, D, device="cuda", generator=g).to(torch.bfloat16)
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    table = lambda pages: torch.tensor([pages], dtype=torch.int32, device="cuda")  # noqa: E731
    w = torch.tensor([100], dtype=torch.int32, device="cuda")
    lmk = torch.tensor([3, 130, 290], dtype=torch.int32, device="cuda").expand(4, 1, 3).contiguous()
    for kw in ({}, dict(w_sizes=w, lmk_indices=lmk)):
        assert torch.equal(V.cache_attention(q, *big, table(ids), lens, **kw),
                           V.cache_attention(q, *small, table([0, 1, 2, 3]), lens, **kw))
    del big
    far = torch.empty((1 << 31) + 2 * 40 * 128, dtype=torch.bfloat16, device="cuda")
    x = far.as_strided((2, 1, 64), (1 << 31, 64, 1))
    x.copy_(torch.randn(2, 1, 64, device="cuda", generator=g))
    caches = [[torch.zeros(2, 1, 16, 64, dtype=torch.uint8, device="cuda").view(F8) for _ in range(2)]
              + [torch.zeros(2, 1, device="cuda") for _ in range(2)] for _ in range(2)]
    at = torch.tensor([0, 16], device="cuda")
    V.append_cache(x, x, *caches[0], at)
    V.append_cache(x.contiguous(), x.contiguous(), *caches[1], at)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    one = torch.tensor([1, 1], dtype=torch.int32, device="cuda")
    tab = torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    assert torch.equal(V.cache_attention(x, *caches[0], tab, one), V.cache_attention(x.contiguous(), *caches[0], tab, one))
    logits = far.as_strided((2, 5000), (1 << 31, 1))
    logits.copy_(torch.randn(2, 5000, device="cuda", generator=g))
    u = torch.tensor([0.3, 0.8], device="cuda")
    for f in ({}, dict(top_k=50), dict(top_p=0.9)):
        assert torch.equal(V.sample_tokens(logits, u, **f), V.sample_tokens(logits.contiguous(), u, **f))
    assert status() == 0


def test_serving_steps_together(V):
    """Admission, prompts, decode steps and release of several requests, each step checked."""
    g = np.random.default_rng(20)
    S, H, Hkv, D, page, n_pages, max_pages = 5, 4, 2, 64, 16, 40, 12
    tg = torch.Generator().manual_seed(20)
    tables = torch.full((S, max_pages), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(S, dtype=torch.int32, device="cuda")
    free = torch.from_numpy(g.permutation(n_pages).astype(np.int32)).cuda()
    n_free = torch.tensor([n_pages], dtype=torch.int32, device="cuda")
    kc = torch.zeros(n_pages, Hkv, page, D, device="cuda").to(F8)
    vc, ks = kc.clone(), torch.zeros(n_pages, Hkv, device="cuda")
    vs = ks.clone()
    rk, rv = (np.zeros((n_pages, Hkv, page, D)), np.zeros((n_pages, Hkv))), (np.zeros((n_pages, Hkv, page, D)), np.zeros((n_pages, Hkv)))
    for step in range(14):
        new = torch.from_numpy(g.integers(0, 50, S).astype(np.int32)) if step in (0, 7) else torch.from_numpy(
            g.integers(0, 3, S).astype(np.int32))
        T = int(new.sum()) + 3  # padded
        plan = V.reserve_slots(tables, lens, new.cuda(), free, n_free, page, T, inplace=True)
        k, v, q = (torch.randn(T, h, D, generator=tg).bfloat16() for h in (Hkv, Hkv, H))
        V.append_cache(k.cuda(), v.cuda(), kc, vc, ks, vs, plan.slots)
        slots = plan.slots.cpu().numpy()
        rk, rv = O.append(k.double().numpy(), *rk, slots, page), O.append(v.double().numpy(), *rv, slots, page)
        np.testing.assert_array_equal(kc.double().cpu().numpy(), rk[0])
        np.testing.assert_array_equal(vs.cpu().numpy(), rv[1])
        granted = plan.granted.cpu().numpy()
        out, lse = V.cache_attention(q.cuda(), kc, vc, ks, vs, tables, lens, cu_q=plan.cu_new, return_lse=True)
        cu = plan.cu_new.cpu().numpy()
        c = dict(q=q[:cu[-1]], kc=rk[0], vc=rv[0], ks=rk[1], vs=rv[1], tables=tables.cpu().numpy(), lens=lens.cpu().numpy(),
                 cu=cu, w=None, lmk=None, bias=None)
        check_attend(c, out[:cu[-1]], lse[:cu[-1]], f"step {step}")
        assert granted.shape == (S,)
        if step in (6, 10):
            V.release_slots(tables, lens, torch.from_numpy(g.random(S) < 0.5).cuda(), free, n_free, page)
    assert status() == 0
