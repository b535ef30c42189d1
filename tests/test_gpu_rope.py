"""tc_rope_turns, tc_rope_apply and tc_rope_kv_write against the same in 64 bits (tests/step.py)."""
import numpy as np
import pytest
import torch

import tc_hip
from paged import TOP, Batch, scaled
from paged import DT as CACHE_DT
from step import DT, HALF, LEAST, f64, rope_exact, tensor, turns_exact

pytestmark = pytest.mark.gpu

RAGGED = [(3, 3), (1, 17), (0, 9), (5, 40), (0, 0), (16, 16), (2, 33)]
SCALINGS = [dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
            dict(scaling="yarn", factor=4.0, original=32768), dict(scaling="yarn", factor=16.0, original=4096, low=2.0, high=40.0),
            dict(scaling="yarn", factor=0.5, original=4096), dict(scaling="yarn", factor=4.0, original=3),
            dict(scaling="bands", factor=8.0, original=8192, low=1.0, high=4.0)]


@pytest.mark.parametrize("kw", SCALINGS, ids=lambda kw: "-".join(str(v) for v in kw.values()) or "none")
@pytest.mark.parametrize("n_rot,theta", [(128, 1e6), (64, 1e4), (4, 10000.0), (250, 5e5)])
def test_turns(dev, n_rot, theta, kw):
    """A power is a few steps of fp64 off, and what is made of it a few more; BANDS and YARN blend with a part that is off
    by some steps of 1: 2^-48 of the larger of both frequencies."""
    r = tc_hip.Rope(n_rot, theta, **kw)
    want, m = turns_exact(n_rot, theta, **kw)
    bound = 2.0 ** -48 * want
    if kw.get("scaling") in ("yarn", "bands"):
        bound = bound * max(kw["factor"], 1 / kw["factor"]) * max(kw["original"], 1.0)
    assert (np.abs(r.turns.cpu().numpy() - want) <= bound).all()
    assert abs(r.c.factor - m) <= 2.0 ** -24 * m
    div = np.linspace(1.0, 3.0, n_rot // 2).astype(np.float32)
    d = tc_hip.Rope(n_rot, theta, divisors=tensor(div, dev), factor_of_values=1.25, **kw)
    assert (np.abs(d.turns.cpu().numpy() * div - r.turns.cpu().numpy()) <= 2.0 ** -50 * want).all()
    assert d.c.factor == 1.25


def near(got, want, err, xtype):
    bad = np.abs(f64(got) - want) > err + HALF[xtype] * (np.abs(want) + err) + LEAST[xtype]
    assert not bad.any(), (np.argwhere(bad)[:4], f64(got)[bad][:4], want[bad][:4], err[bad][:4])


@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("xtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("heads,dim,n_rot", [(1, 16, 16), (5, 80, 80), (3, 96, 48), (28, 128, 128), (2, 128, 2), (7, 128, 90),
                                             (4, 256, 250), (2, 192, 64)])
def test_apply(tc, dev, heads, dim, n_rot, xtype, layout):
    """Positions near and far, below 0 (left alone), odd numbers of pairs, parts of a head, rows at a stride, in place."""
    rng = np.random.default_rng(dim + n_rot)
    pos = np.array([0, 1, 2, 7, 131071, -1, 1000003, 5, 2 ** 26, -2 ** 31, 12345], np.int32)
    T = len(pos)
    rope = tc_hip.Rope(n_rot, 1e6, layout=layout, factor_of_values=1.25)
    wide = torch.from_numpy(rng.standard_normal((T, heads + 2, dim)).astype(np.float32)).to(DT[xtype]).to(dev)
    x = wide[:, 1:1 + heads]
    # (at 2^26 the product with the fp64 frequency and that itself are off by 2^-53 of 2^23.3 turns)
    want, err = rope_exact(f64(x), pos, turns_exact(n_rot, 1e6)[0], n_rot, layout, 1.25)
    err += np.abs(f64(x)).max() * 2 * 1.25 * np.maximum(pos, 0)[:, None, None] * 2.0 ** -52
    want[pos < 0], err[pos < 0] = f64(x)[pos < 0], 0
    out = torch.full((T, heads, dim), 7.0, dtype=DT[xtype], device=dev)
    given = tensor(pos, dev)
    assert tc.rope(rope, x, given, out=out) is out
    assert (out[pos < 0] == 7.0).all()
    new = tc.rope(rope, x, given)
    near(new, want, err, xtype)
    live = torch.from_numpy(pos >= 0).to(dev)
    assert torch.equal(out[live], new[live])
    whole = wide.clone()
    tc.rope(rope, whole[:, 1:1 + heads], given, out=whole[:, 1:1 + heads])  # in place, the neighbours untouched
    assert torch.equal(whole[:, 1:1 + heads], new)
    assert torch.equal(whole[:, 0], wide[:, 0]) and torch.equal(whole[:, 1 + heads:], wide[:, 1 + heads:])


def test_apply_long(tc, dev):
    """Enough rows for lanes that have four heads each, heads that four does not divide."""
    rng = np.random.default_rng(1)
    pos = rng.integers(0, 200000, 4001).astype(np.int32)
    x = torch.from_numpy(rng.standard_normal((4001, 18, 64)).astype(np.float32)).to(dev)
    rope = tc_hip.Rope(64, 1e4)
    want, err = rope_exact(f64(x), pos, turns_exact(64, 1e4)[0], 64, "half", 1.0)
    near(tc.rope(rope, x, tensor(pos, dev)), want, err, "F32")
    assert tc.rope(rope, x[:0], tensor(pos[:0], dev)).shape == (0, 18, 64)


def test_turn_keeps_lengths(tc, dev):
    """Scores depend on the distance alone: q at p + d with k at p, in fp32, for p from 0 to 10^6."""
    rng = np.random.default_rng(2)
    rope = tc_hip.Rope(128, 1e6, layout="pairs")
    q, k = (torch.from_numpy(np.repeat(rng.standard_normal((1, 1, 128)), 8, 0).astype(np.float32)).to(dev) for _ in range(2))
    p = np.array([0, 1, 17, 1000, 65536, 131071, 999999, 1000000], np.int32)
    a, b = f64(tc.rope(rope, q, tensor(p + 37, dev))), f64(tc.rope(rope, k, tensor(p, dev)))
    s = (a * b).sum((1, 2))
    # each rotated value is off by 5 roundings of its pair's magnitudes
    bound = 2 * 5 * 2.0 ** -24 * 2 * (np.abs(f64(q)).max() + 1) * np.abs(f64(k)).sum(2).max() + 1e-12
    assert np.abs(s - s[0]).max() <= bound


def setup(rng, dev, xtype, ctype, heads, kv, dim, page, seqs=RAGGED, pad=2):
    b = Batch(rng, seqs, page, kv, dim, ctype, pad_rows=pad).to(dev)
    x = rng.standard_normal((b.T, heads + 2 * kv, dim)) * np.exp(rng.standard_normal((1, heads + 2 * kv, 1)))
    x = torch.from_numpy(x.astype(np.float32)).to(DT[xtype]).to(dev)
    return b, x, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]


CTYPES = ["F16", "BF16", "I8", "E4M3"]


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("xtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("layout,heads,kv,dim,page,n_rot", [("half", 28, 4, 128, 16, 128), ("pairs", 3, 1, 80, 48, 40),
                                                            ("half", 6, 3, 96, 32, 90), ("pairs", 2, 2, 256, 64, 256),
                                                            ("half", 4, 4, 48, 16, 16)])
def test_kv_write(tc, dev, layout, heads, kv, dim, page, n_rot, xtype, ctype, norms):
    """Queries, cached keys and values of every row; every other slot and row as it was."""
    rng = np.random.default_rng(dim + heads)
    b, x, q, k, v = setup(rng, dev, xtype, ctype, heads, kv, dim, page)
    rope = tc_hip.Rope(n_rot, 1e6, layout=layout, scaling="yarn", factor=4.0, original=64)
    turns, m = turns_exact(n_rot, 1e6, scaling="yarn", factor=4.0, original=64)
    w = [1 + 0.3 * rng.standard_normal(dim).astype(np.float32) if norms else None for _ in range(2)]
    dw = [None if a is None else tensor(a, dev) for a in w]
    before = {n: t.clone() for n, t in b.dev.items()}
    out = torch.full((b.T, heads, dim), 7.0, dtype=DT[xtype], device=dev)
    assert tc.rope_kv_write(b.cache, b.batch, rope, q, k, v, q_norm=dw[0], k_norm=dw[1], eps=1e-5, out=out) is out
    rows = list(b.rows())
    pos = np.zeros(b.T, np.int64)
    pos[[t for t, _, _ in rows]] = [p for _, _, p in rows]
    live = np.zeros(b.T, bool)
    live[[t for t, _, _ in rows]] = True
    want, err = rope_exact(f64(q), pos, turns, n_rot, layout, float(np.float32(m)), w[0], 1e-5)
    near(out[torch.from_numpy(live)], want[live], err[live], xtype)
    assert (out[torch.from_numpy(~live)] == 7.0).all()
    kw, kerr = rope_exact(f64(k), pos, turns, n_rot, layout, float(np.float32(m)), w[1], 1e-5)
    for name, val, err in (("k", kw, kerr), ("v", f64(v), np.zeros_like(kw))):
        got, old = b.dev[name].float().cpu().numpy().astype(np.float64), before[name].float().cpu().numpy()
        sc = b.dev[name + "_scale"].double().cpu().numpy() if scaled(ctype) else None
        touched = np.zeros(got.shape[:1] + got.shape[2:3], bool)
        for t, s, p in rows:
            at = b.slot(s, p)
            if at is None:
                continue
            touched[at] = True
            have = got[at[0], :, at[1]]
            if sc is None:
                half = HALF[ctype] * (np.abs(val[t]) + err[t]) + LEAST[ctype]
            else:
                # the factor's and the quotient's roundings, then half a step of the 8-bit number
                d = np.abs(val[t]).max(-1, keepdims=True) / TOP[ctype]
                have = have * sc[at[0], :, at[1]][:, None]
                step = d / 2 if ctype == "I8" else np.maximum(2.0 ** -4 * np.abs(val[t]), 2.0 ** -10 * d)
                half = step * 1.001 + 3 * 2.0 ** -24 * np.abs(val[t]) + 2 * err[t].max(-1, keepdims=True)
            assert (np.abs(have - val[t]) <= err[t] + half).all(), (name, t)
        keep = ~touched[:, None, :].repeat(kv, 1)
        assert np.array_equal(got[keep], old[keep])
        if sc is not None:
            assert np.array_equal(sc[keep], before[name + "_scale"].double().cpu().numpy()[keep])


@pytest.mark.parametrize("ctype", CTYPES)
@pytest.mark.parametrize("layout", ["half", "pairs"])
@pytest.mark.parametrize("seqs", [RAGGED, [(1, 40)], [(700, 900), (1, 5), (350, 350)], [(k % 4, 5 + k % 37) for k in range(300)]],
                         ids=["ragged", "one", "long", "many"])
def test_fused_is_the_parts(tc, dev, seqs, layout, ctype):
    """fp32 rows: rotating, then tc_kv_write, gives the same bits in the cache and the queries."""
    rng = np.random.default_rng(len(seqs))
    b, x, q, k, v = setup(rng, dev, "F32", ctype, 8, 4, 128, 32, seqs)
    rope = tc_hip.Rope(96, 1e6, layout=layout)
    start = {n: t.clone() for n, t in b.dev.items()}
    out = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v)
    fused = {n: t.clone() for n, t in b.dev.items()}
    for n, t in b.dev.items():
        t.copy_(start[n])
    pos = torch.full((b.T,), -1, dtype=torch.int32)
    for t, s, p in b.rows():
        pos[t] = p
    pos = pos.to(dev)
    tc.kv_write(b.cache, b.batch, tc.rope(rope, k, pos), v.contiguous())
    for n, t in b.dev.items():
        assert torch.equal(t.view(torch.uint8), fused[n].view(torch.uint8)), n
    live = pos >= 0
    assert torch.equal(out[live], tc.rope(rope, q, pos)[live])


def test_in_place_and_keys_alone(tc, dev):
    rng = np.random.default_rng(5)
    b, x, q, k, v = setup(rng, dev, "BF16", "F16", 6, 2, 64, 16)
    rope = tc_hip.Rope(64)
    out = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v)
    held = {n: t.clone() for n, t in b.dev.items()}
    qc = q.contiguous()
    tc.rope_kv_write(b.cache, b.batch, rope, qc, k, v, out=qc)
    live = int(b.start[-1])
    assert torch.equal(qc[:live], out[:live]) and torch.equal(qc[live:], q[live:])
    # in place among the rows of one product: keys, values and padding as they were
    whole = x.clone()
    part = whole[:, :6]
    assert tc.rope_kv_write(b.cache, b.batch, rope, part, whole[:, 6:8], whole[:, 8:], out=part) is part
    assert torch.equal(whole[:live, :6], out[:live]) and torch.equal(whole[live:], x[live:]) and torch.equal(whole[:, 6:], x[:, 6:])
    assert all(torch.equal(t, held[n]) for n, t in b.dev.items())
    for bad in (whole[:, 1:7], whole.view(-1)[:b.T * 6 * 64].view(b.T, 6, 64), out[:, :5], out.float()):
        with pytest.raises(tc_hip.TCError):
            tc.rope_kv_write(b.cache, b.batch, rope, part, whole[:, 6:8], whole[:, 8:], out=bad)
    for t in b.dev.values():
        t.zero_()
    assert tc.rope_kv_write(b.cache, b.batch, rope, None, k, v) is None
    for t, s, p in b.rows():
        if b.slot(s, p):
            pg, sl = b.slot(s, p)
            assert torch.equal(b.dev["k"][pg, :, sl], held["k"][pg, :, sl])


def test_many_heads(tc, dev):
    """More heads than a model has: units of a token over many workgroups."""
    rng = np.random.default_rng(8)
    b, x, q, k, v = setup(rng, dev, "BF16", "I8", 1000, 20, 32, 16, seqs=[(2, 20), (1, 1)], pad=0)
    rope = tc_hip.Rope(32, layout="pairs")
    out = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v)
    want, err = rope_exact(f64(q), np.array([18, 19, 0]), turns_exact(32, 1e4)[0], 32, "pairs", 1.0)
    near(out, want, err, "BF16")
    got = tc.kv_read(b.cache, b.batch, 3, torch.float32)[0]
    want, err = rope_exact(f64(k), np.array([18, 19, 0]), turns_exact(32, 1e4)[0], 32, "pairs", 1.0)
    step = np.abs(want).max(-1, keepdims=True) / 127 / 2
    assert (np.abs(f64(got) - want) <= step * 1.001 + 2 * err.max(-1, keepdims=True) + 3 * 2.0 ** -24 * np.abs(want)).all()


def test_rows_without_slots(tc, dev):
    """Pages that the table has not or that do not exist: queries are rotated all the same, nothing else is written."""
    rng = np.random.default_rng(6)
    b, x, q, k, v = setup(rng, dev, "F32", "I8", 4, 2, 64, 16, seqs=[(20, 40), (5, 5)], pad=0)
    rope = tc_hip.Rope(64)
    want = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v)
    table = b.batch.table
    table[0, 2] = -1
    table[1, 0] = b.n_pages
    before = {n: t.clone() for n, t in b.dev.items()}
    for n, t in b.dev.items():
        t.zero_()
    zero = {n: t.clone() for n, t in b.dev.items()}
    out = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v)
    assert torch.equal(out, want)
    for n, t in b.dev.items():
        changed = (t != zero[n]).reshape(b.n_pages, 2, 16, -1).any(-1).any(1)
        assert int(changed.sum()) == 12, n  # positions 20 to 31 of the first sequence
    del before


def test_extreme_rows(tc, dev):
    """Infinities and NaN stay in their row; rows of zeros get the factor 1; fp16's largest."""
    rng = np.random.default_rng(7)
    b, x, q, k, v = setup(rng, dev, "F16", "E4M3", 2, 2, 64, 16, seqs=[(6, 6)], pad=0)
    x[0, 2, 3], x[1, 0, 5], x[2, 3, 0] = float("inf"), float("nan"), float("-inf")
    x[3] = 0
    x[4] = 65504.0
    rope = tc_hip.Rope(64)
    out = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v, q_norm=torch.ones(64, device=dev), k_norm=torch.ones(64, device=dev))
    assert not torch.isfinite(out[1, 0]).all() and torch.isfinite(out[1, 1]).all() and torch.isfinite(out[[0, 2, 3, 4, 5]]).all()
    pg, ks = int(b.table[0, 0]), b.dev["k_scale"]
    assert (ks[pg, :, 3] == 1.0).all() and (b.dev["v_scale"][pg, :, 3] == 1.0).all()
    kv = tc.kv_read(b.cache, b.batch, b.T, torch.float32)[0]
    assert not torch.isfinite(kv[0, 0]).any() and not torch.isfinite(kv[2, 1]).any()
    assert torch.isfinite(kv[[1, 3, 4, 5]]).all() and torch.isfinite(kv[0, 1]).all()


# a prompt and sequences around it: enough rows that a lane has four heads, five and three of which leave some lanes fewer
PROMPTS = [(1900, 1900), (1, 70), (0, 5), (160, 333), (3, 3)]


@pytest.mark.parametrize("norms", [False, True])
@pytest.mark.parametrize("ctype", ["F16", "BF16", "E4M3", "I8"])
@pytest.mark.parametrize("xtype", ["F16", "BF16", "F32"])
@pytest.mark.parametrize("layout,dim,n_rot", [("half", 128, 128), ("half", 128, 90), ("pairs", 128, 64), ("half", 80, 48),
                                              ("pairs", 256, 250)])
def test_prompts(tc, dev, layout, dim, n_rot, xtype, ctype, norms):
    """Prompts' rows: queries in place among the rows of one product, cached keys and values; the rest as it was."""
    rng = np.random.default_rng(dim + n_rot)
    heads, kv, page = 5, 3, 32
    b, x, q, k, v = setup(rng, dev, xtype, ctype, heads, kv, dim, page, PROMPTS, pad=3)
    # (four heads a lane from 1024 workgroups of 256 lanes with one head each)
    lanes = 16 if dim <= 128 else 32
    assert b.T * (heads + 2 * kv) * lanes > 1200 * 256
    rope = tc_hip.Rope(n_rot, 1e6, layout=layout, factor_of_values=1.25)
    turns, _ = turns_exact(n_rot, 1e6)
    w = [1 + 0.3 * rng.standard_normal(dim).astype(np.float32) if norms else None for _ in range(2)]
    dw = [None if a is None else tensor(a, dev) for a in w]
    before = {n: t.clone() for n, t in b.dev.items()}
    given = x.clone()
    assert tc.rope_kv_write(b.cache, b.batch, rope, q, k, v, q_norm=dw[0], k_norm=dw[1], eps=1e-5, out=q) is q
    T = int(b.start[-1])
    assert torch.equal(x[:, heads:], given[:, heads:]) and torch.equal(x[T:], given[T:])
    pos = np.array([p for _, _, p in b.rows()])
    page_of, place = (np.array(a) for a in zip(*(b.slot(s, p) for _, s, p in b.rows())))
    want, err = rope_exact(f64(given[:T, :heads]), pos, turns, n_rot, layout, 1.25, w[0], 1e-5)
    near(x[:T, :heads], want, err, xtype)
    val, off = rope_exact(f64(given[:T, heads:heads + kv]), pos, turns, n_rot, layout, 1.25, w[1], 1e-5)
    for name, val, off in (("k", val, off), ("v", f64(given[:T, heads + kv:]), np.zeros_like(val))):
        got, old = (t[name].float().cpu().numpy().astype(np.float64) for t in (b.dev, before))
        have = got[page_of, :, place]
        if scaled(ctype):
            # the factor's and the quotient's roundings, then half a step of the 8-bit number
            have = have * f64(b.dev[name + "_scale"])[page_of, :, place][..., None]
            d = np.abs(val).max(-1, keepdims=True) / TOP[ctype]
            step = d / 2 if ctype == "I8" else np.maximum(2.0 ** -4 * np.abs(val), 2.0 ** -10 * d)
            half = step * 1.001 + 3 * 2.0 ** -24 * np.abs(val) + 2 * off.max(-1, keepdims=True)
        else:
            half = HALF[ctype] * (np.abs(val) + off) + LEAST[ctype]
        bad = np.abs(have - val) > off + half
        assert not bad.any(), (name, np.argwhere(bad)[:4], have[bad][:4], val[bad][:4])
        touched = np.zeros(got.shape[:1] + got.shape[2:3], bool)
        touched[page_of, place] = True
        keep = ~touched[:, None, :].repeat(kv, 1)
        assert np.array_equal(got[keep], old[keep])
        if scaled(ctype):
            assert np.array_equal(f64(b.dev[name + "_scale"])[keep], f64(before[name + "_scale"])[keep])


@pytest.mark.parametrize("layout,n_rot", [("half", 128), ("half", 122), ("pairs", 128)])
@pytest.mark.parametrize("xtype", ["F16", "BF16", "F32"])
def test_apply_prompts(tc, dev, xtype, layout, n_rot):
    """Rows at positions, four heads a lane, in place at a stride."""
    rng = np.random.default_rng(n_rot)
    T, heads = 2500, 9
    pos = rng.integers(-3, 200000, T).astype(np.int32)
    pos[::7] = -1
    wide = torch.from_numpy(rng.standard_normal((T, heads + 1, 128)).astype(np.float32)).to(DT[xtype]).to(dev)
    before = wide.clone()
    rope = tc_hip.Rope(n_rot, 1e6, layout=layout)
    tc.rope(rope, wide[:, :heads], tensor(pos, dev), out=wide[:, :heads])
    assert torch.equal(wide[:, heads], before[:, heads])
    given = f64(before[:, :heads])
    want, err = rope_exact(given, pos, turns_exact(n_rot, 1e6)[0], n_rot, layout, 1.0)
    # (at 2 10^5 the product with the fp64 frequency and that itself are off by 2^-53 of 2^15 turns)
    err += np.abs(given).max() * 2 * np.maximum(pos, 0)[:, None, None] * 2.0 ** -52
    want[pos < 0], err[pos < 0] = given[pos < 0], 0
    near(wide[:, :heads], want, err, xtype)


def test_head_norms_near_the_range(tc, dev):
    """Squares of values around 10^18 and 10^-18, without eps."""
    rng = np.random.default_rng(9)
    for dim in (64, 256):
        b, x, q, k, v = setup(rng, dev, "F32", "BF16", 3, 1, dim, 16, seqs=[(9, 9)], pad=0)
        for size in (1e18, 1e-18):
            sign = np.where(rng.random((9, 3, dim)) < 0.5, -1.0, 1.0)
            q.copy_(tensor((size * sign).astype(np.float32), dev))
            rope = tc_hip.Rope(dim, 1e4)
            out = tc.rope_kv_write(b.cache, b.batch, rope, q, k, v, q_norm=torch.ones(dim, device=dev), eps=0.0)
            want, err = rope_exact(f64(q), np.arange(9), turns_exact(dim, 1e4)[0], dim, "half", 1.0, np.ones(dim), 0.0)
            near(out, want, err, "F32")
