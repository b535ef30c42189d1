"""CPU tests of the cache, attention and verification entry points: refusals,
and the geometry of a batch whose arrays hold anything at all."""
import ctypes

import pytest
import torch

import tc_hip
from test_capi import _compile_and_run


@pytest.fixture(scope="module")
def lib():
    return tc_hip.load_library()


BUF = ctypes.create_string_buffer(1 << 12)
P = (ctypes.addressof(BUF) + 255) & ~255  # (an address; nothing on the CPU reads it)


def cache(**kw):
    f = dict(type=tc_hip.F16, n_pages=4, kv_heads=2, page_tokens=16, head_dim=64, k=P, v=P, k_scale=None, v_scale=None)
    f.update(kw)
    return tc_hip._CKVCache(**f)


def batch(**kw):
    f = dict(n_seq=1, n_tokens=2, table_pages=3, start=P, len=P, table=P)
    f.update(kw)
    return tc_hip._CKVBatch(**f)


def write(lib, c, b, xtype=0, k=P, v=P, ks=128, vs=128):
    return lib.tc_kv_write(ctypes.byref(c) if c else None, ctypes.byref(b) if b else None, xtype, k, v, ks, vs, None)


def attn(lib, c, b, xtype=0, q=P, qs=256, out=P, heads=4, scale=0.125, window=0):
    return lib.tc_attn(ctypes.byref(c), ctypes.byref(b), xtype, q, qs, out, heads, scale, window, None)


ARG, UNSUPPORTED = tc_hip.TC_E_ARG, tc_hip.TC_E_UNSUPPORTED
I8 = dict(type=tc_hip.I8, k_scale=P, v_scale=P)


@pytest.mark.parametrize("c,b,code,word", [
    (dict(type=8), {}, UNSUPPORTED, "cache type"),
    (dict(k=None), {}, ARG, "null"),
    (dict(v=None), {}, ARG, "null"),
    (dict(type=tc_hip.I8), {}, ARG, "scales"),
    (dict(type=tc_hip.E4M3, k_scale=P), {}, ARG, "scales"),
    (dict(k_scale=P, v_scale=P), {}, ARG, "scales"),
    (dict(head_dim=72), {}, UNSUPPORTED, "head_dim"),
    (dict(head_dim=272), {}, UNSUPPORTED, "head_dim"),
    (dict(head_dim=0), {}, UNSUPPORTED, "empty"),
    (dict(page_tokens=24), {}, UNSUPPORTED, "page_tokens"),
    (dict(page_tokens=0), {}, UNSUPPORTED, "empty"),
    (dict(n_pages=0), {}, UNSUPPORTED, "empty"),
    (dict(kv_heads=0), {}, UNSUPPORTED, "empty"),
    (dict(k=P + 8), {}, UNSUPPORTED, "aligned"),
    (dict(I8, v_scale=P + 2), {}, UNSUPPORTED, "aligned"),
    (dict(n_pages=1 << 31), {}, UNSUPPORTED, "pages"),
    ({}, dict(start=None), ARG, "null"),
    ({}, dict(len=None), ARG, "null"),
    ({}, dict(table=None), ARG, "null"),
    ({}, dict(table=P + 1), UNSUPPORTED, "aligned"),
    ({}, dict(table_pages=0), UNSUPPORTED, "empty"),
    ({}, dict(n_tokens=(1 << 24) + 1), UNSUPPORTED, "rows"),
    ({}, dict(n_seq=(1 << 20) + 1), UNSUPPORTED, "sequences"),
])
def test_cache_and_batch_refusals(lib, c, b, code, word):
    for rc in (write(lib, cache(**c), batch(**b)), attn(lib, cache(**c), batch(**b)),
               lib.tc_kv_read(ctypes.byref(cache(**c)), ctypes.byref(batch(**b)), 0, P, P, None)):
        assert rc == code
        assert word in lib.tc_last_error().decode()


def test_row_refusals(lib):
    assert write(lib, None, batch()) == ARG and write(lib, cache(), None) == ARG
    assert write(lib, cache(), batch(), xtype=tc_hip.I8) == UNSUPPORTED
    assert write(lib, cache(), batch(), k=None) == ARG
    assert write(lib, cache(), batch(), ks=127) == ARG  # rows that overlap
    assert write(lib, cache(), batch(), vs=130) == UNSUPPORTED  # fp32 rows at 8-byte distances
    assert write(lib, cache(), batch(), xtype=tc_hip.F16, vs=132) == UNSUPPORTED
    assert write(lib, cache(), batch(), k=P + 4) == UNSUPPORTED
    assert attn(lib, cache(), batch(), heads=3) == UNSUPPORTED
    assert attn(lib, cache(), batch(), heads=0) == UNSUPPORTED
    assert attn(lib, cache(), batch(), qs=255) == ARG
    assert attn(lib, cache(), batch(), out=None) == ARG
    assert attn(lib, cache(), batch(), out=P + 8) == UNSUPPORTED
    for bad in (float("nan"), float("inf"), -0.5):
        assert attn(lib, cache(), batch(), scale=bad) == ARG
    # nothing to do is done anywhere
    assert attn(lib, cache(), batch(n_tokens=0)) == tc_hip.TC_OK
    assert write(lib, cache(), batch(n_seq=0)) == tc_hip.TC_OK


def verify(lib, **kw):
    f = dict(logits=P, probs=None, vocab=100, n_seq=1, n_tokens=2, start=P, tokens=P, temperature=P, accept=P, sample=P,
             n=P, token=P, stream=None)
    f.update(kw)
    return lib.tc_spec_verify(*f.values())


def test_verify_refusals(lib):
    for name in ("logits", "start", "tokens", "temperature", "accept", "sample", "n", "token"):
        assert verify(lib, **{name: None}) == ARG
        assert verify(lib, **{name: P + 2}) == UNSUPPORTED
    assert verify(lib, vocab=0) == UNSUPPORTED and verify(lib, vocab=(1 << 30) + 1) == UNSUPPORTED
    assert verify(lib, n_tokens=65536) == UNSUPPORTED and verify(lib, n_seq=65536) == UNSUPPORTED
    assert verify(lib, n_tokens=0) == UNSUPPORTED
    assert verify(lib, n_seq=0) == tc_hip.TC_OK


def test_without_a_device(lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for rc in (write(lib, cache(), batch()), attn(lib, cache(**I8), batch()), verify(lib), lib.tc_attn_reserve(8, 8)):
        assert rc == UNSUPPORTED and b"gfx950" in lib.tc_last_error()


def test_binding_refusals():
    """What the Python classes check before a call."""
    f16 = torch.zeros(2, 1, 16, 32, dtype=torch.float16)
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVCache(f16, f16.to(torch.bfloat16))
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVCache(f16, f16, torch.zeros(2, 1, 16), torch.zeros(2, 1, 16))
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVCache(f16.to(torch.int8), f16.to(torch.int8))
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVCache(f16[:, :, :, ::2], f16[:, :, :, ::2])
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVCache(f16.double(), f16.double())
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVBatch(i, i[:2].long(), torch.zeros(2, 4, dtype=torch.int32))
    with pytest.raises(tc_hip.TCError):
        tc_hip.KVBatch(i, i, torch.zeros(3, 4, dtype=torch.int32))


def test_geometry_of_any_arrays(tmp_path):
    """Random start, len and table arrays, most of them nonsense: every row range stays in the call's rows,
    every cache row in the cache, and the sound ones are where the definition puts them (run under the address
    sanitizer, with the arrays at their exact sizes)."""
    _compile_and_run(tmp_path, r"""
#include <stdio.h>
#include <stdlib.h>
#include <random>
#include <vector>
#include "tc_kv_index.hpp"
int main() {
    std::mt19937 rng(1);
    auto r = [&](int64_t lo, int64_t hi) { return lo + int64_t(rng() % uint64_t(hi - lo + 1)); };
    for (int turn = 0; turn < 3000; ++turn) {
        tc::KvArgs a{};
        a.n_seq = uint32_t(r(1, 9));
        a.n_tokens = uint32_t(r(1, 40));
        a.table_pages = uint32_t(r(1, 6));
        a.n_pages = uint32_t(r(1, 12));
        a.kv_heads = uint32_t(r(1, 5));
        a.page = uint32_t(16 * r(1, 9));
        a.page_div = tc::make_divmod(a.page);
        const bool wild = turn % 2;
        std::vector<int32_t> start(a.n_seq + 1), len(a.n_seq), table(size_t(a.n_seq) * a.table_pages);
        for (uint32_t s = 0; s <= a.n_seq; ++s) start[s] = wild ? int32_t(rng()) >> int(r(0, 28)) : s == 0 ? 0 : int32_t(r(start[s - 1], a.n_tokens));
        for (auto &x : len) x = wild ? int32_t(rng()) >> int(r(0, 28)) : int32_t(r(0, 6 * 150));
        for (auto &x : table) x = wild ? int32_t(rng()) >> int(r(0, 28)) : int32_t(r(-1, a.n_pages));
        a.start = start.data(); a.len = len.data(); a.table = table.data();
        const int64_t rows = int64_t(a.n_pages) * a.kv_heads * a.page;
        for (uint32_t s = 0; s < a.n_seq; ++s) {
            uint32_t b, e;
            tc::seq_rows(a.start, a.n_tokens, s, &b, &e);
            if (b > e || e > a.n_tokens) return printf("rows %u %u\n", b, e), 1;
        }
        for (uint32_t t = 0; t < a.n_tokens; ++t) {
            const int s = tc::find_seq(a.start, a.n_seq, t);
            if (s < -1 || s >= int(a.n_seq)) return printf("sequence %d\n", s), 1;
            for (uint32_t h = 0; h < a.kv_heads; ++h) {
                const int64_t x = tc::slot_of(a, s, t, h);
                if (x < -1 || x >= rows) return printf("row %lld\n", (long long)x), 1;
                if (wild) continue;
                int64_t want = -1;
                for (uint32_t q = 0; q < a.n_seq; ++q) {
                    if (int(t) < start[q] || int(t) >= start[q + 1]) continue;
                    const int64_t pos = len[q] - start[q + 1] + int(t);
                    if (pos < 0 || pos / a.page >= a.table_pages) continue;
                    const int32_t pg = table[q * a.table_pages + pos / a.page];
                    if (pg >= 0 && pg < int(a.n_pages)) want = (int64_t(pg) * a.kv_heads + h) * a.page + pos % a.page;
                }
                if (x != want) return printf("row %lld, not %lld\n", (long long)x, (long long)want), 1;
            }
        }
    }
    return 0;
}
""", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined")


def test_binding_refuses_numbers_beyond_32_bits():
    """What ctypes would cut to 32 bits."""
    tc = tc_hip.Library()
    c = tc_hip.KVCache(*(torch.zeros(2, 1, 16, 32, dtype=torch.float16) for _ in range(2)))
    b = tc_hip.KVBatch(*(torch.zeros(s, dtype=torch.int32) for s in ((2,), (1,), (1, 2))))
    q = torch.zeros(1, 1, 32)
    for window in (-1, 1 << 32):
        with pytest.raises(tc_hip.TCError, match="window"):
            tc.attn(c, b, q, 1.0, window=window)
    for args in ((-1, 4), (4, -1), (1 << 32, 1), (8, 1 << 32)):
        with pytest.raises(tc_hip.TCError, match="32 bits"):
            tc.attn_reserve(*args)
    far = torch.empty_strided((2, 1, 32), ((1 << 32) + 64, 32, 1), device="meta")
    with pytest.raises(tc_hip.TCError, match="32 bits"):
        tc._row_stride(far)
    assert tc._row_stride(far[:1]) == 32 and tc._row_stride(torch.empty(2, 3, 32, device="meta")) == 96


def test_batch_of_no_sequences(lib):
    """Arrays without an entry have no address: a call for no sequences does nothing, and says so."""
    none = batch(n_seq=0, n_tokens=0, len=None, table=None)
    padded = batch(n_seq=0, len=None, table=None)
    for b in (none, padded):
        assert write(lib, cache(), b) == tc_hip.TC_OK
        assert attn(lib, cache(), b) == tc_hip.TC_OK
        assert lib.tc_kv_read(ctypes.byref(cache()), ctypes.byref(b), 0, P, P, None) == tc_hip.TC_OK
    assert write(lib, cache(), batch(n_seq=0, start=None, len=None, table=None)) == ARG
