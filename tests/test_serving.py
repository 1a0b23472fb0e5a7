"""Serving operators without a GPU: their oracle against independent statements of the same
definitions, and the refusals of the C ABI and of the torch-facing functions."""
import ctypes
import os

import numpy as np
import pytest
import torch

from dsalt_b200 import _lib as L
from dsalt_b200 import serving as V
from oracle import serving_oracle as O


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(L.LIB_PATH):
        from dsalt_b200 import build
        build.build()
    return L.load()


# ------------------------------------------------------------------ the oracle itself
def test_oracle_e4m3_equals_torchs_cast():
    bits = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(bits, O.VALUES)
    x = torch.cat([torch.randn(20000) * 2.0 ** torch.randint(-14, 9, (20000,)), torch.tensor([0.0, -0.0, 448.0])])
    x = torch.cat([x, torch.from_numpy((O.VALUES[:126] + O.VALUES[1:127]) / 2).float()])  # ties
    ref = x.clamp(-448, 448).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(O.to_e4m3(x.double().numpy()), ref)


@pytest.mark.parametrize("amax,e", [(448.0, 0), (448.5, 1), (224.0, -1), (1.0, -8), (1.75, -8), (1.7500001, -7),
                                    (3.0e38, 120), (1e-38, O.E_MIN), (0.0, O.E_MIN)])
def test_oracle_scale_exponent(amax, e):
    assert O.need_exponent(amax) == e
    if amax and e > O.E_MIN:
        assert amax <= 448 * 2.0 ** e and amax > 448 * 2.0 ** (e - 1)


def test_oracle_reserve_never_gives_a_page_twice():
    g = np.random.default_rng(0)
    S, page, max_pages, n_pages = 7, 16, 9, 40
    tables, lens = np.full((S, max_pages), -1, np.int32), np.zeros(S, np.int32)
    free, n_free = g.permutation(n_pages).astype(np.int32), n_pages
    for _ in range(60):
        new = g.integers(0, 40, S)
        tables, slots, _, cu, granted, lens, n_free = O.reserve(tables, lens, new, free, n_free, page, 400)
        owned = tables[tables >= 0]
        assert len(set(owned)) == len(owned) and set(owned).isdisjoint(free[:n_free])
        assert len(owned) + n_free == n_pages
        used = slots[slots >= 0]
        assert len(set(used)) == len(used) and len(used) == sum(min(int(x), 400) for x in new[granted])
        flags = g.random(S) < 0.3
        tables, lens, free, n_free = O.release(tables, lens, flags, free, n_free, page)


def test_oracle_sample_without_filters_is_the_inverse_of_the_distribution():
    g = np.random.default_rng(1)
    l = g.normal(size=50)
    p = np.exp(l) / np.exp(l).sum()
    draws = [O.sample(l, (i + 0.5) / 20000, 1.0, 0, 1.0, 0.0)[0] for i in range(20000)]
    # equally spaced uniforms: each token's count is its probability to within one spacing
    assert np.abs(np.bincount(draws, minlength=50) / 20000 - p).max() <= 1 / 20000 + 1e-12
    assert O.sample(l, 0.3, 0.0, 0, 1.0, 0.0)[0] == int(l.argmax())
    assert O.sample(l, 0.99, 1.0, 1, 1.0, 0.0)[0] == int(l.argmax())
    assert O.sample(l, 0.99, 1.0, 0, 0.0, 0.0)[0] == int(l.argmax())


# ------------------------------------------------------------------ refusals of the C ABI
FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below fails before device work


def test_slots_arguments_are_rejected(lib):
    def reserve(S=4, max_pages=8, cap=32, page=16, n=8, tables=FAKE, slots=FAKE, granted=FAKE):
        return lib.dsalt_reserve_slots(tables, S, max_pages, FAKE, FAKE, FAKE, cap, FAKE, page, n, slots, FAKE, FAKE,
                                       granted, FAKE, FAKE, None)

    assert reserve(S=0) == L.ERR_INVALID and reserve(n=-1) == L.ERR_INVALID and reserve(cap=-1) == L.ERR_INVALID
    assert reserve(page=24) == L.ERR_UNSUPPORTED and b"page size 24" in lib.dsalt_last_error()
    assert reserve(S=V.MAX_ROWS + 1) == L.ERR_UNSUPPORTED and reserve(n=1 << 31) == L.ERR_UNSUPPORTED
    assert reserve(tables=None) == L.ERR_INVALID and reserve(granted=None) == L.ERR_INVALID
    assert reserve(slots=None) == L.ERR_INVALID and b"null pointer" in lib.dsalt_last_error()
    assert reserve(slots=ctypes.c_void_p(4100)) == L.ERR_INVALID and b"aligned" in lib.dsalt_last_error()

    def release(S=4, page=16, flags=FAKE):
        return lib.dsalt_release_slots(FAKE, S, 8, FAKE, flags, FAKE, 32, FAKE, page, None)

    assert release(S=0) == L.ERR_INVALID and release(page=0) == L.ERR_UNSUPPORTED
    assert release(S=V.MAX_ROWS + 1) == L.ERR_UNSUPPORTED and release(flags=None) == L.ERR_INVALID


def test_append_arguments_are_rejected(lib):
    def append(k=FAKE, dtype=L.BF16, T=8, n_kv=2, D=64, ts=128, hs=64, pages=4, page=16, slots=FAKE, scale=FAKE):
        return lib.dsalt_append_cache(k, FAKE, dtype, T, n_kv, D, ts, hs, ts, hs, FAKE, FAKE, scale, FAKE, pages, page,
                                      slots, None)

    assert append(T=-1) == L.ERR_INVALID and append(n_kv=0) == L.ERR_INVALID and append(pages=-1) == L.ERR_INVALID
    assert append(dtype=7) == L.ERR_INVALID
    assert append(D=96) == L.ERR_UNSUPPORTED and append(page=48) == L.ERR_UNSUPPORTED
    assert append(k=None) == L.ERR_INVALID and append(slots=None) == L.ERR_INVALID
    assert append(scale=None) == L.ERR_INVALID
    assert append(k=ctypes.c_void_p(4098)) == L.ERR_INVALID and append(ts=129) == L.ERR_INVALID
    assert append(T=0, k=None, slots=None) == L.OK  # nothing to do


def test_cache_attention_arguments_are_rejected(lib):
    need = lib.dsalt_cache_attention_workspace_bytes(8, 8, 4, 2, 64)
    assert need > 0 and need % 256 == 0
    assert lib.dsalt_cache_attention_workspace_bytes(8, 0, 4, 2, 64) == 0

    def attend(q=FAKE, dtype=L.BF16, T=8, H=4, Hkv=2, D=64, qs=256, pages=4, page=16, max_pages=4, S=8, cu=None, w=FAKE,
               lmk=FAKE, k=3, out=FAKE, odt=L.BF16, ws=FAKE, ws_bytes=need):
        return lib.dsalt_cache_attention(q, dtype, T, H, Hkv, D, qs, FAKE, FAKE, FAKE, FAKE, pages, page, FAKE, max_pages,
                                         FAKE, S, cu, w, lmk, None, k, out, odt, None, ws, ws_bytes, None)

    assert attend(H=3) == L.ERR_INVALID and attend(S=0, T=0) == L.ERR_INVALID and attend(k=-1) == L.ERR_INVALID
    assert attend(max_pages=0) == L.ERR_INVALID and attend(T=-1) == L.ERR_INVALID
    assert attend(dtype=5) == L.ERR_INVALID and attend(odt=5) == L.ERR_INVALID
    assert attend(D=32, qs=256) == L.ERR_UNSUPPORTED and attend(page=8) == L.ERR_UNSUPPORTED
    assert attend(T=9) == L.ERR_INVALID and b"one query per sequence" in lib.dsalt_last_error()
    assert attend(qs=255) == L.ERR_INVALID and attend(qs=260) == L.ERR_INVALID
    assert attend(w=None) == L.ERR_INVALID and b"window widths" in lib.dsalt_last_error()
    assert attend(q=None) == L.ERR_INVALID and attend(out=None) == L.ERR_INVALID and attend(lmk=None) == L.ERR_INVALID
    assert attend(ws=None) == L.ERR_INVALID
    assert attend(ws_bytes=need - 256) == L.ERR_WORKSPACE
    assert attend(pages=1 << 27, page=128) == L.ERR_UNSUPPORTED
    assert attend(S=V.MAX_ROWS + 1, T=V.MAX_ROWS + 1) == L.ERR_UNSUPPORTED
    assert attend(T=0, q=None, ws=None, cu=FAKE) == L.OK


def test_sample_arguments_are_rejected(lib):
    def sample(logits=FAKE, dtype=L.F32, B=2, Vn=100, stride=100, u=FAKE, token=FAKE):
        return lib.dsalt_sample(logits, dtype, B, Vn, stride, u, None, 1.0, None, 0, None, 1.0, None, 0.0, token, None,
                                None)

    assert sample(B=-1) == L.ERR_INVALID and sample(Vn=0) == L.ERR_INVALID and sample(stride=99) == L.ERR_INVALID
    assert sample(dtype=4) == L.ERR_INVALID
    assert sample(Vn=V.MAX_VOCAB + 1, stride=V.MAX_VOCAB + 1) == L.ERR_UNSUPPORTED
    assert sample(logits=None) == L.ERR_INVALID and sample(u=None) == L.ERR_INVALID and sample(token=None) == L.ERR_INVALID
    assert sample(logits=ctypes.c_void_p(4098)) == L.ERR_INVALID
    assert sample(B=0, logits=None, u=None, token=None) == L.OK


# ------------------------------------------------------------------ refusals of the torch-facing functions
def test_cpu_tensors_are_rejected():
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    f8 = torch.zeros(2, 2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = torch.ones(2, 2)
    with pytest.raises(RuntimeError, match="no CPU path"):
        V.reserve_slots(i32(2, 4), i32(2), i32(2), i32(8), i32(1), 16, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        V.release_slots(i32(2, 4), i32(2), torch.zeros(2, dtype=torch.bool), i32(8), i32(1), 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        V.append_cache(torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), f8, f8, sc, sc, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        V.cache_attention(torch.zeros(2, 2, 64), f8, f8, sc, sc, i32(2, 4), i32(2))
    with pytest.raises(RuntimeError, match="no CPU path"):
        V.sample_tokens(torch.zeros(2, 10), torch.zeros(2))


def test_settings_are_checked():
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            V._setting(bad, "temperature", 1, torch.float32, 0.0, 3e38)
    with pytest.raises(ValueError):
        V._setting(1.5, "min_p", 1, torch.float32, 0.0, 1.0)
    with pytest.raises(TypeError):
        V._setting(torch.zeros(2, dtype=torch.float64), "top_p", 2, torch.float32, 0.0, 1.0)
    with pytest.raises(ValueError):
        V._setting(torch.zeros(3), "top_p", 2, torch.float32, 0.0, 1.0)
    assert V._setting(0.5, "top_p", 2, torch.float32, 0.0, 1.0) == (None, 0.5)
