"""The paged cache (tc_kv_write, tc_kv_read) and attention over it (tc_attn)
against the same in 64 bits (tests/paged.py)."""
import ctypes

import numpy as np
import pytest
import torch

from paged import DT, HALF, TOP, Batch, attn_bound, attn_exact, scaled

pytestmark = pytest.mark.gpu

XTYPES, CTYPES = ["F32", "F16", "BF16"], ["F16", "BF16", "I8", "E4M3"]
# (new rows, length): from the first token, appended, none new, an empty sequence, over page borders
RAGGED = [(3, 3), (1, 17), (0, 9), (5, 40), (0, 0), (16, 16), (2, 33)]


def rows_of(rng, T, heads, dim, xtype, spread=1.0):
    return torch.from_numpy((spread * rng.standard_normal((T, heads, dim))).astype(np.float32)).to(DT[xtype])


# ---- write and read ---------------------------------------------------------------------------------------------


def written(b, name, x):
    """The cache after tc_kv_write of x: (values as held, scales), numpy fp32."""
    held = b.host[name].float().numpy().copy()
    sc = b.host[name + "_scale"].numpy().copy() if scaled(b.ctype) else None
    x = x.float().numpy()
    for t, s, pos in b.rows():
        w = b.slot(s, pos)
        if w is None:
            continue
        r = x[t]
        if sc is not None:
            d = (np.abs(r).max(-1) / np.float32(TOP[b.ctype])).astype(np.float32)
            d[d == 0] = 1
            sc[w[0], :, w[1]] = d
            r = (r / d[:, None]).astype(np.float32)
            r = np.rint(r) if b.ctype == "I8" else torch.from_numpy(r).to(DT["E4M3"]).float().numpy()
        else:
            r = torch.from_numpy(r).to(DT[b.ctype]).float().numpy()
        held[w[0], :, w[1]] = r
    return held, sc


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("xtype", XTYPES)
@pytest.mark.parametrize("kv_heads,dim,page", [(4, 128, 16), (1, 16, 48), (3, 80, 32), (2, 256, 64)])
def test_kv_write(tc, dev, xtype, ctype, kv_heads, dim, page):
    """Every slot of the batch holds its row's values and every other one what it held; ties, rows of zeros,
    large and small rows."""
    rng = np.random.default_rng(dim + page)
    b = Batch(rng, RAGGED, page, kv_heads, dim, ctype, pad_rows=2)
    k, v = (rows_of(rng, b.T, kv_heads, dim, xtype) for _ in range(2))
    k[0] = 0
    k[1, :, :4] = torch.tensor([127.0, 0.5, 2.5, -1.5])  # halves of steps where the scale is 1
    k[1, :, 4:] = 3.5
    v[2] *= 1e4
    v[3] *= 1e-4
    b.to(dev)
    tc.kv_write(b.cache, b.batch, k.to(dev), v.to(dev))
    for name, x in (("k", k), ("v", v)):
        held, sc = written(b, name, x)
        assert np.array_equal(b.dev[name].float().cpu().numpy(), held), name
        if sc is not None:
            assert np.array_equal(b.dev[name + "_scale"].cpu().numpy(), sc), name


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("xtype", XTYPES)
@pytest.mark.parametrize("kv_heads,dim,page", [(4, 128, 16), (1, 48, 48), (3, 112, 32)])
def test_kv_read(tc, dev, xtype, ctype, kv_heads, dim, page):
    """Rows come back as value * scale, rounded once; rows past the last sequence are left alone."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, RAGGED, page, kv_heads, dim, ctype, pad_rows=3).to(dev)
    out = tuple(torch.full((b.T, kv_heads, dim), 7.0, dtype=DT[xtype], device=dev) for _ in range(2))
    tc.kv_read(b.cache, b.batch, b.T, DT[xtype], out=out)
    for name, got in zip(("k", "v"), out):
        want = np.full((b.T, kv_heads, dim), 7.0)
        value = b.value(name)
        for t, s, pos in b.rows():
            p, i = b.slot(s, pos)
            want[t] = value[p, :, i]
        got = got.double().cpu().numpy()
        # value * scale is rounded to fp32 and then to the rows' type
        err = np.abs(got - want)
        assert (err <= np.abs(want) * (HALF[xtype] * 1.001 + 2.0 ** -24) + 2.0 ** -25).all(), (name, err.max())
        assert (got[-3:] == 7).all()


@pytest.mark.parametrize("n_seq", [63, 64, 65, 5000])
@pytest.mark.parametrize("ctype", ["BF16", "I8"])
def test_kv_many_sequences(tc, dev, ctype, n_seq):
    """Sequences of no, one and several rows: each row into its own pages and back, more of them than one lane takes."""
    rng = np.random.default_rng(n_seq)
    new = rng.choice([0, 0, 1, 1, 2, 17], n_seq)
    seqs = [(int(n), int(n + rng.integers(0, 40))) for n in new]
    b = Batch(rng, seqs, 16, 2, 48, ctype, pad_rows=3).to(dev)
    k, v = (rows_of(rng, b.T, 2, 48, "F32") for _ in range(2))
    tc.kv_write(b.cache, b.batch, k.to(dev), v.to(dev))
    got = [t.cpu() for t in tc.kv_read(b.cache, b.batch, b.T, torch.float32,
                                       out=tuple(torch.full((b.T, 2, 48), 7.0, device=dev) for _ in range(2)))]
    used = int(b.start[-1])
    for x, y in zip((k, v), got):
        # bf16: half a step; int8: half a step of max / 127, and the two roundings of the quotients and of the product
        top = x.abs().amax(-1, keepdim=True)
        bound = x.abs() * 2.0 ** -8 if ctype == "BF16" else top / 127 * 0.5 + x.abs() * 2.0 ** -22
        assert ((x - y).abs() <= bound)[:used].all() and (y[used:] == 7).all()


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
def test_kv_write_extremes(tc, dev, ctype):
    """A row with an infinity or a NaN reads back as NaNs, its neighbours do not; a row of the smallest
    numbers reads back within a step of it."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [(4, 20)], 16, 2, 64, ctype).to(dev)
    k = rows_of(rng, 4, 2, 64, "F32")
    v = k.clone()
    k[0, 0, 5], k[1, 1, 7], k[2, 0, 63] = float("inf"), float("nan"), float("-inf")
    v[3] = 1e-44
    tc.kv_write(b.cache, b.batch, k.to(dev), v.to(dev))
    rk, rv = (x.cpu() for x in tc.kv_read(b.cache, b.batch, 4, torch.float32))
    bad = torch.zeros(4, 2, dtype=torch.bool)
    bad[0, 0] = bad[1, 1] = bad[2, 0] = True
    assert torch.equal(rk.isnan().all(-1), bad) and torch.equal(rk.isnan().any(-1), bad)
    assert (rv[3].abs() <= 2e-44).all()


def test_kv_strided_rows(tc, dev):
    """q, k and v as parts of one fused product's rows."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [(5, 21), (1, 4)], 16, 2, 64, "F16").to(dev)
    rows = rows_of(rng, 6, 8, 64, "F32").to(dev)  # 4 query heads, 2 of keys, 2 of values
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    tc.kv_write(b.cache, b.batch, k, v)
    got = tc.attn(b.cache, b.batch, q, 0.125)
    for name, x in (("k", k), ("v", v)):
        assert np.array_equal(b.dev[name].float().cpu().numpy(), written(b, name, x.cpu())[0])
    assert torch.equal(got, tc.attn(b.cache, b.batch, q.contiguous(), 0.125))


# ---- attention ---------------------------------------------------------------------------------------------------


def check_attn(tc, dev, b, heads, xtype, scale, window=0, spread=1.0, seed=0):
    rng = np.random.default_rng(seed)
    q = rows_of(rng, b.T, heads, b.dim, xtype, spread)
    out = torch.full((b.T, heads, b.dim), 7.0, dtype=DT[xtype], device=dev)
    tc.attn(b.cache, b.batch, q.to(dev), scale, window=window, out=out)
    got = out.double().cpu().numpy()
    want, mass, terms, absv = attn_exact(b, q.double().numpy(), scale, window)
    n = max(total for _, total in b.seqs)
    bound = attn_bound(xtype, b.ctype, b.dim, n, want, mass, terms, absv)
    used = int(b.start[-1])
    err = np.abs(got - want)[:used]
    worst = (err / bound[:used]).max() if used else 0
    assert (got[used:] == 7).all()
    assert not (worst > 1) and np.isfinite(got).all(), worst
    return got, bound


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("xtype", XTYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 4, 64, 16), (14, 2, 128, 32), (8, 1, 256, 48), (3, 3, 80, 16), (6, 2, 16, 64)])
def test_attn_ragged(tc, dev, xtype, ctype, heads, kv_heads, dim, page):
    rng = np.random.default_rng(heads + dim)
    b = Batch(rng, RAGGED, page, kv_heads, dim, ctype, pad_rows=2).to(dev)
    check_attn(tc, dev, b, heads, xtype, dim ** -0.5)


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("xtype", XTYPES)
def test_attn_decode_lengths(tc, dev, xtype, ctype):
    """One token each at lengths around every tile and page border."""
    rng = np.random.default_rng(1)
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 47, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 1025]
    b = Batch(rng, [(1, n) for n in lens], 16, 2, 64, ctype).to(dev)
    check_attn(tc, dev, b, 6, xtype, 0.125)


@pytest.mark.parametrize("ctype,xtype,dim", [("BF16", "BF16", 128), ("F16", "F32", 128), ("I8", "F16", 64), ("E4M3", "BF16", 256),
                                             ("BF16", "F32", 96), ("I8", "F32", 256), ("F16", "F16", 192), ("BF16", "F16", 64)])
@pytest.mark.parametrize("n,total", [(130, 130), (65, 400), (257, 300), (40, 1000)])
def test_attn_prompts(tc, dev, ctype, xtype, dim, n, total):
    rng = np.random.default_rng(n)
    b = Batch(rng, [(n, total), (1, 70), (9, 9)], 32, 2, dim, ctype).to(dev)
    check_attn(tc, dev, b, 6, xtype, dim ** -0.5)


@pytest.mark.parametrize("window", [1, 7, 16, 33, 64, 100, 4096])
@pytest.mark.parametrize("ctype,xtype", [("F16", "F32"), ("E4M3", "BF16"), ("BF16", "BF16")])
def test_attn_window(tc, dev, window, ctype, xtype):
    rng = np.random.default_rng(window)
    b = Batch(rng, [(1, 300), (150, 200), (5, 64), (3, 3), (30, 95)], 16, 2, 64, ctype).to(dev)
    check_attn(tc, dev, b, 8, xtype, 0.125, window=window)


@pytest.mark.parametrize("xtype", XTYPES)
@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("spread,scale", [(60.0, 0.125), (1e-6, 0.125), (1.0, 0.0)])
def test_attn_sharp_and_flat(tc, dev, xtype, ctype, spread, scale):
    """Softmaxes of one token, and flat ones."""
    rng = np.random.default_rng(2)
    b = Batch(rng, [(1, 200), (70, 90)], 16, 1, 64, ctype).to(dev)
    check_attn(tc, dev, b, 4, xtype, scale, spread=spread)


def test_attn_large_and_small_values(tc, dev):
    """Rows of q far outside fp16's range, and factors of very different sizes."""
    rng = np.random.default_rng(3)
    b = Batch(rng, [(1, 100), (40, 60)], 16, 1, 64, "I8")
    b.host["v_scale"] *= torch.from_numpy(np.exp2(rng.integers(-40, 40, b.host["v_scale"].shape)).astype(np.float32))
    b.host["k_scale"] *= 2.0 ** -20
    b.to(dev)
    check_attn(tc, dev, b, 4, "F32", 0.125, spread=2.0 ** 20)
    check_attn(tc, dev, b, 4, "BF16", 0.125, spread=2.0 ** 20)
    b = Batch(rng, [(1, 100), (40, 60)], 16, 1, 64, "BF16")
    for name in ("k", "v"):
        b.host[name] *= 2.0 ** 40
    b.to(dev)
    check_attn(tc, dev, b, 4, "F32", 2.0 ** -43)


def test_attn_rows_that_see_nothing(tc, dev):
    """Rows at positions below 0 (more new rows than tokens), and sequences whose pages are all missing, give
    zeros; a missing page among others is skipped, and so is what lies past the table."""
    rng = np.random.default_rng(4)
    b = Batch(rng, [(5, 2), (1, 40), (3, 50), (1, 0), (2, 100)], 16, 2, 64, "F16", width=4)
    b.table[1, :] = -1
    b.table[2, 1] = b.n_pages
    b.to(dev)
    got, _ = check_attn(tc, dev, b, 4, "F32", 0.125)
    assert (got[:3] == 0).all() and (got[5] == 0).all() and (got[9] == 0).all()
    k = rows_of(rng, b.T, 2, 64, "F32")
    tc.kv_write(b.cache, b.batch, k.to(dev), k.to(dev))
    for name in ("k", "v"):
        assert np.array_equal(b.dev[name].float().cpu().numpy(), written(b, name, k)[0])
    rk, _ = tc.kv_read(b.cache, b.batch, b.T, torch.float32)
    for t, s, pos in b.rows():
        if b.slot(s, pos) is None:
            assert (rk[t] == 0).all()


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("n", [2, 120])
def test_attn_table_ends_inside_a_tile(tc, dev, ctype, n):
    """Lengths past what the table has room for, which ends in the middle of 32 tokens; a page missing between others."""
    rng = np.random.default_rng(11)
    b = Batch(rng, [(n, 200), (n, 190), (n, 150)], 16, 1, 64, ctype, width=5)
    b.table[1, 2] = -1
    b.table[2, 1:3] = b.n_pages + 7
    check_attn(tc, dev, b.to(dev), 4, "F32", 0.125)


@pytest.mark.parametrize("n_seq", [511, 512, 513, 1300])
def test_attn_many_sequences(tc, dev, n_seq):
    """Sequences of no, one and several rows among many; two of them prompts."""
    rng = np.random.default_rng(n_seq)
    new = rng.choice([0, 1, 1, 1, 3], n_seq)
    new[[2, n_seq - 1]] = 40, 36
    seqs = [(int(n), int(n + rng.integers(0, 30))) for n in new]
    b = Batch(rng, seqs, 16, 2, 32, "F16", pad_rows=3).to(dev)
    check_attn(tc, dev, b, 4, "F32", 0.2)
    none = Batch(rng, [(0, 5)] * n_seq, 16, 2, 32, "F16", pad_rows=4).to(dev)
    check_attn(tc, dev, none, 4, "F32", 0.2)


@pytest.mark.parametrize("ctype,xtype", [("BF16", "BF16"), ("F16", "F32"), ("I8", "F32"), ("E4M3", "F16")])
@pytest.mark.parametrize("dim", [48, 64, 112, 128, 208, 240])
def test_attn_block_borders(tc, dev, ctype, xtype, dim):
    """As many rows as fill blocks of either kind, one less and one more, alone in a head and in groups."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, [(n, n + int(rng.integers(0, 80))) for n in (15, 16, 17, 63, 64, 65, 127, 129)], 48, 1, dim, ctype).to(dev)
    check_attn(tc, dev, b, 1, xtype, dim ** -0.5)
    b = Batch(rng, [(n, n + int(rng.integers(0, 80))) for n in (5, 6, 21, 22, 43, 86)], 16, 1, dim, ctype, pad_rows=1).to(dev)
    check_attn(tc, dev, b, 3, xtype, dim ** -0.5, window=40)


@pytest.mark.parametrize("group", [1, 5, 64, 65, 300])
def test_attn_groups(tc, dev, group):
    """Groups as large as the blocks of rows and larger: a token's rows lie in several blocks."""
    rng = np.random.default_rng(group)
    b = Batch(rng, [(1, 33), (2, 50), (7, 7)], 16, 2, 32, "BF16").to(dev)
    check_attn(tc, dev, b, 2 * group, "BF16", 0.2)


def test_attn_captured_at_first(tc, dev):
    """The first call of its kind, captured after tc_attn_reserve alone."""
    rng = np.random.default_rng(13)
    b = Batch(rng, [(1, 90), (40, 70)], 32, 2, 144, "E4M3").to(dev)
    q = rows_of(rng, b.T, 4, 144, "F32").to(dev)
    tc.attn_reserve(4, b.T)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tc.attn(b.cache, b.batch, q, 0.1)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, tc.attn(b.cache, b.batch, q, 0.1))


def test_attn_batch_of_several_calls(tc, dev):
    """One batch for calls of different numbers of rows, as a program's padded and whole steps make them."""
    rng = np.random.default_rng(14)
    b = Batch(rng, [(1, 40), (2, 30)], 16, 2, 64, "F16", pad_rows=5).to(dev)
    q = rows_of(rng, b.T, 4, 64, "F32").to(dev)
    whole = tc.attn(b.cache, b.batch, q, 0.125)
    assert torch.equal(tc.attn(b.cache, b.batch, q[:3].contiguous(), 0.125), whole[:3])
    k, _ = tc.kv_read(b.cache, b.batch, 3, torch.float32)
    assert torch.equal(tc.kv_read(b.cache, b.batch, 3, torch.float32)[0], k)
    assert torch.equal(tc.attn(b.cache, b.batch, q, 0.125)[:3], whole[:3])


@pytest.mark.parametrize("ctype", ["F16", "I8"])
@pytest.mark.parametrize("n", [1, 80])
def test_attn_long_parts(tc, dev, ctype, n):
    """As many heads as there are compute units, so that each takes thousands of tokens."""
    rng = np.random.default_rng(12)
    H, D, total = 256, 16, 20001
    b = Batch(rng, [(n, total)], 48, H, D, ctype).to(dev)
    q = rows_of(rng, n, H, D, "F32")
    got = tc.attn(b.cache, b.batch, q.to(dev), 0.25).double().cpu().numpy()
    at = np.arange(total)
    pg, sl = torch.from_numpy(b.table[0, at // 48].astype(np.int64)).to(dev), torch.from_numpy(at % 48).to(dev)
    seen = torch.arange(total, device=dev)[None] <= torch.arange(total - n, total, device=dev)[:, None]
    for h in range(0, H, 37):
        k, v = (b.dev[x][pg, h, sl].double() for x in ("k", "v"))
        if ctype == "I8":
            k, v = (x * b.dev[c][pg, h, sl].double()[:, None] for x, c in ((k, "k_scale"), (v, "v_scale")))
        x = q[:, h].double().to(dev)
        p = torch.softmax((x @ k.T * 0.25).masked_fill(~seen, float("-inf")), 1)
        absv = seen.double() @ v.abs()
        terms = (x.abs() @ k.abs().T * 0.25).masked_fill(~seen, 0).amax(1, keepdim=True)
        want, mass, absv, terms = (y.cpu().numpy() for y in (p @ v, p @ v.abs(), absv, terms))
        assert (np.abs(got[:, h] - want) <= attn_bound("F32", ctype, D, total, want, mass, terms, absv)).all(), h


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("n", [1, 3, 70])
def test_attn_ignores_what_it_does_not_see(tc, dev, ctype, n):
    """Infinities and NaN behind a sequence's end, in free pages and in tokens that a row does not see change
    nothing."""
    rng = np.random.default_rng(7)
    b = Batch(rng, [(n, 90), (1, 37)], 32, 2, 64, ctype)
    clean, bound = check_attn(tc, dev, b.to(dev), 6, "F32", 0.125, window=50)
    used = {b.slot(s, j) for s, (_, total) in enumerate(b.seqs) for j in range(total)}
    bad = torch.ones(b.n_pages, b.page, dtype=torch.bool)
    for p, i in used:
        bad[p, i] = False
    # the last row of the first sequence is seen by itself alone
    last = b.slot(0, 89)
    for name in ("k", "v"):
        h = b.host[name]
        for p, i in [(int(p), int(i)) for p, i in bad.nonzero()] + [last]:
            if scaled(ctype):
                b.host[name + "_scale"][p, :, i] = float("nan") if (p + i) % 2 else float("inf")
                if ctype == "E4M3":
                    h.view(torch.uint8)[p, :, i] = 0x7F
            else:
                h[p, :, i] = float("nan") if (p + i) % 2 else float("inf")
    b.to(dev)
    q = rows_of(np.random.default_rng(0), b.T, 6, 64, "F32")
    got = tc.attn(b.cache, b.batch, q.to(dev), 0.125, window=50).double().cpu().numpy()
    rest = np.arange(n + 1) != n - 1
    assert (np.abs(got - clean)[rest] <= 2 * bound[rest]).all()
    assert np.isnan(got[n - 1]).any()


def test_attn_shared_pages(tc, dev):
    """Sequences that share their first pages."""
    rng = np.random.default_rng(8)
    b = Batch(rng, [(1, 70), (4, 68), (90, 150)], 16, 2, 64, "BF16")
    b.table[1, :4] = b.table[0, :4]
    b.table[2, :3] = b.table[0, :3]
    check_attn(tc, dev, b.to(dev), 4, "BF16", 0.125)


def test_attn_step_as_a_graph(tc, dev):
    """Write, attention and read of a chunk captured once and replayed with other lengths, pages and rows:
    every replay gives the eager calls' bits, with eager work of other sizes between the replays."""
    rng = np.random.default_rng(9)
    sizes = [[(1, 70), (3, 33), (60, 61)], [(1, 500), (0, 0), (63, 200)], [(2, 2), (60, 90), (2, 3)]]
    steps = [Batch(rng, s, 16, 2, 64, "I8", spare=40 - sum(-(-t // 16) for _, t in s) + 40, width=40) for s in sizes]
    live = Batch(rng, sizes[0], 16, 2, 64, "I8", spare=80 - 11, width=40).to(dev)
    other = Batch(rng, [(1, 3000)], 16, 4, 128, "F16").to(dev)
    T = 64
    q = torch.zeros(T, 8, 64, device=dev)
    kv = torch.zeros(2, T, 2, 64, device=dev)
    tc.attn_reserve(8, T)

    def work():
        tc.kv_write(live.cache, live.batch, kv[0], kv[1])
        o = tc.attn(live.cache, live.batch, q, 0.125)
        return o, *tc.kv_read(live.cache, live.batch, T, torch.float32)

    work()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = work()
    for turn in range(2):
        for b in steps:
            for name, t in b.host.items():
                live.dev[name].zero_()
                live.dev[name][:t.shape[0]] = t.to(dev)[:live.n_pages]
            live.batch.start.copy_(torch.from_numpy(b.start))
            live.batch.length.copy_(torch.from_numpy(b.length))
            live.batch.table.copy_(torch.from_numpy(b.table))
            q.copy_(rows_of(rng, T, 8, 64, "F32"))
            kv.copy_(rows_of(rng, 2 * T, 2, 64, "F32").reshape(2, T, 2, 64))
            for o in outs:
                o.fill_(3.0)
            tc.attn(other.cache, other.batch, torch.randn(1, 8, 128, device=dev), 0.1)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            got = [o[:b.start[-1]].clone() for o in outs]
            want = [o[:b.start[-1]] for o in work()]
            for x, y in zip(got, want):
                assert torch.equal(x, y), (turn, b.seqs)


def test_attn_on_another_stream(tc, dev):
    rng = np.random.default_rng(10)
    b = Batch(rng, [(1, 900), (40, 300)], 16, 2, 128, "BF16").to(dev)
    q = rows_of(rng, b.T, 14, 128, "BF16").to(dev)
    want = tc.attn(b.cache, b.batch, q, 0.09)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = tc.attn(b.cache, b.batch, q, 0.09)
    s.synchronize()
    assert torch.equal(got, want)


def test_attn_cache_beyond_4_gib(tc, dev):
    """Pages whose bytes lie past 32-bit offsets."""
    page, kvh, dim = 1024, 8, 256
    n_pages = (9 << 30) // (page * kvh * dim * 2)
    k, v = (torch.zeros(n_pages, kvh, page, dim, dtype=torch.bfloat16, device=dev) for _ in range(2))
    import tc_hip
    cache = tc_hip.KVCache(k, v)
    g = torch.Generator().manual_seed(0)
    table = torch.tensor([[n_pages - 1, 1, n_pages - 2]], dtype=torch.int32, device=dev)
    batch = tc_hip.KVBatch(torch.tensor([0, 2500], dtype=torch.int32, device=dev),
                           torch.tensor([2500], dtype=torch.int32, device=dev), table)
    rows = [torch.randn(2500, kvh, dim, generator=g).to(torch.bfloat16) for _ in range(2)]
    tc.kv_write(cache, batch, *(r.to(dev) for r in rows))
    back = tc.kv_read(cache, batch, 2500, torch.bfloat16)
    for x, y in zip(rows, back):
        assert torch.equal(x, y.cpu())
    assert int((k != 0).any(-1).sum()) == 2500 * kvh
    q = torch.randn(1, 8, dim, generator=g).to(torch.bfloat16)
    one = tc_hip.KVBatch(torch.tensor([0, 1], dtype=torch.int32, device=dev), batch.length, table)
    got = tc.attn(cache, one, q.to(dev), 0.0625).double().cpu()
    kd, vd = (r.double() for r in rows)
    for h in range(8):
        p = torch.softmax(kd[:, h] @ q[0, h].double() * 0.0625, 0)
        want, mass = p @ vd[:, h], p @ vd[:, h].abs()
        assert ((got[0, h] - want).abs() <= mass * (2.0 ** -8 + 2e-3) + 2.0 ** -8 * want.abs()).all()


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
@pytest.mark.parametrize("factor", [0.0, 2.0 ** -126, 2.0 ** -118])
@pytest.mark.parametrize("size", [1.0, 100.0])
def test_attn_next_to_no_values(tc, dev, ctype, factor, size):
    """Tokens whose values are nothing beside the others', as in slots of a fresh cache (factors of 0) that a length
    reaches: their weights count in the sum, small ones too."""
    rng = np.random.default_rng(24)
    b = Batch(rng, [(1, 400), (70, 200), (4, 100)], 16, 2, 64, ctype)
    b.host["v_scale"] *= size
    at = torch.from_numpy(rng.random(b.host["v_scale"].shape) < 0.5)
    b.host["v_scale"][at] = factor
    if factor == 0:
        for name in ("k", "v"):
            b.host[name].view(torch.uint8)[at] = 0
        b.host["k_scale"][at] = 0
    b.to(dev)
    for spread in (1.0, 5.0, 9.0):
        check_attn(tc, dev, b, 4, "F32", 0.125, spread=spread)


def zero_rows(b, rng, share, factor):
    """Makes rows of values zeros (of either sign where there are two), with this factor; -> which."""
    at = torch.from_numpy(rng.random(b.host["v_scale"].shape) < share)
    v = b.host["v"].view(torch.uint8)
    v[at] = 0
    if b.ctype == "E4M3":
        v[at & torch.from_numpy(rng.random(at.shape) < 0.5)] = 0x80
    b.host["v_scale"][at] = factor
    return at


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
@pytest.mark.parametrize("xtype", XTYPES)
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 1e-8, 1e-10])
@pytest.mark.parametrize("dim", [64, 112, 256])
def test_attn_rows_of_zeros_among_small_values(tc, dev, ctype, xtype, size, dim):
    """Rows of zeros, to which tc_kv_write gives the factor 1, take nothing of the other rows' precision."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, [(1, 200), (5, 60), (90, 200), (1, 3)], 16, 2, dim, ctype)
    b.host["v_scale"] *= size
    zero_rows(b, rng, 0.05, 1.0)
    check_attn(tc, dev, b.to(dev), 4, xtype, dim ** -0.5)


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
def test_attn_rows_of_zeros_alone(tc, dev, ctype):
    """Sequences that see rows of zeros first, last, in whole tiles, and nothing else."""
    rng = np.random.default_rng(21)
    b = Batch(rng, [(1, 600), (80, 300), (1, 70), (40, 90)], 16, 2, 64, ctype)
    b.host["v_scale"] *= 1e-6
    v, sc = b.host["v"].view(torch.uint8), b.host["v_scale"]
    for s, blocks in ((0, range(0, 20)), (1, range(5, 18)), (2, range(5)), (3, range(6))):
        for i in blocks:
            v[int(b.table[s, i])] = 0
            sc[int(b.table[s, i])] = 1
    got, _ = check_attn(tc, dev, b.to(dev), 4, "F32", 0.125)
    assert (got[81] == 0).all() and (got[82:] == 0).all()


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
@pytest.mark.parametrize("xtype", ["F32", "BF16"])
def test_attn_factors_of_one(tc, dev, ctype, xtype):
    """Rows of values whose factor is 1 and which are not zeros, beside some which are."""
    rng = np.random.default_rng(22)
    b = Batch(rng, [(1, 200), (90, 200)], 16, 2, 64, ctype)
    at = torch.from_numpy(rng.random(b.host["v_scale"].shape) < 0.5)
    b.host["v_scale"][at] = 1
    zero_rows(b, rng, 0.1, 1.0)
    b.host["v"].view(torch.uint8)[:, :, 3, 1:] = 0  # (one value of a row is enough)
    b.host["v_scale"][:, :, 3] = 1
    check_attn(tc, dev, b.to(dev), 4, xtype, 0.125)


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
def test_attn_written_zeros(tc, dev, ctype):
    """Rows of zeros as tc_kv_write leaves them, through the whole path."""
    rng = np.random.default_rng(23)
    b = Batch(rng, [(100, 100), (64, 64)], 16, 2, 64, ctype)
    b.to(dev)
    k, v = rows_of(rng, b.T, 2, 64, "F32"), rows_of(rng, b.T, 2, 64, "F32", 1e-7)
    v[::7] = 0
    v[3::11] = -0.0
    tc.kv_write(b.cache, b.batch, k.to(dev), v.to(dev))
    for name in b.host:
        b.host[name] = b.dev[name].cpu()
    check_attn(tc, dev, b, 4, "F32", 0.125)


@pytest.mark.parametrize("ctype,xtype", [("BF16", "BF16"), ("F16", "F16"), ("F16", "BF16")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attn_of_values_all_alike(tc, dev, ctype, xtype, dim):
    """Weights whose sum is not that of the weights that the values were multiplied with would not give them back."""
    rng = np.random.default_rng(dim)
    b = Batch(rng, [(1, 2), (1, 40), (1, 300), (3, 33), (40, 70), (130, 200), (1, 64), (9, 500)], 16, 2, dim, ctype)
    value = torch.from_numpy(rng.integers(-8, 9, (1, 2, 1, dim)) / 8).to(DT[ctype])
    b.host["v"] = value.expand(b.host["v"].shape).contiguous()
    b.to(dev)
    q = rows_of(rng, b.T, 6, dim, xtype, 2.0)
    got = tc.attn(b.cache, b.batch, q.to(dev), dim ** -0.5).float().cpu()
    want = value.float().reshape(1, 2, 1, dim).expand(b.T, 2, 3, dim).reshape(b.T, 6, dim)
    # (fp32 sums of 500 terms in two orders: 500 * 2^-24, a fraction of half a step of either type)
    assert torch.equal(got, want), (got - want).abs().max()


@pytest.mark.parametrize("ctype", ["I8", "E4M3"])
@pytest.mark.parametrize("xtype", XTYPES)
def test_kv_read_roundings(tc, dev, ctype, xtype):
    """value * scale rounded to fp32, and that to the rows' type: bit for bit."""
    rng = np.random.default_rng(31)
    b = Batch(rng, [(300, 300), (37, 90)], 16, 3, 96, ctype).to(dev)
    got = tc.kv_read(b.cache, b.batch, b.T, DT[xtype])
    at = [b.slot(s, pos) for _, s, pos in b.rows()]
    pg, sl = (torch.tensor(x) for x in zip(*at))
    for name, x in zip(("k", "v"), got):
        want = (b.host[name].float() * b.host[name + "_scale"][..., None])[pg, :, sl].to(DT[xtype])
        assert torch.equal(x.cpu(), want)
