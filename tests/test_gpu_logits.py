"""tc_logits_adjust against the same in 64 bits (tests/step.py)."""
import numpy as np
import pytest
import torch

import tc_hip
from step import DT, f64, logits_exact, tensor

pytestmark = pytest.mark.gpu


def make(rng, V, rows, hist, bias=0, masks=0, drafts=True, xtype="F32"):
    """Rules of sequences of rows[s] rows and hist[s] tokens before them; tokens that come more than once."""
    S, T = len(rows), sum(rows)
    sums = lambda v: np.concatenate([[0], np.cumsum(v)]).astype(np.int32)  # noqa: E731
    few = lambda n: np.minimum((V * rng.random(n) ** 3).astype(np.int32), V - 1)  # noqa: E731
    r = dict(repetition=(0.8 + 0.6 * rng.random(S)).astype(np.float32), frequency=(rng.random(S) - 0.3).astype(np.float32),
             presence=(rng.random(S) - 0.3).astype(np.float32), history=few(sum(hist)), history_start=sums(hist),
             prompt=(rng.random(S) * (np.array(hist) + 2)).astype(np.int32))
    if bias:
        n = rng.integers(0, bias + 1, S)
        r.update(bias_start=sums(n), bias_token=few(int(n.sum())), bias_value=(3 * rng.standard_normal(int(n.sum()))).astype(np.float32))
    if masks:
        r.update(mask=rng.integers(-2 ** 31, 2 ** 31, (masks, (V + 31) // 32)).astype(np.int32),
                 mask_of=rng.integers(-1, masks, T).astype(np.int32))
    l = torch.from_numpy((3 * rng.standard_normal((T, V))).astype(np.float32)).to(DT[xtype])
    return r, l, sums(rows), few(T) if drafts else None


def rules(r, dev):
    return tc_hip.LogitRules(**{k: tensor(v, dev) for k, v in r.items()})


def close(got, want):
    """A changed logit is formed in fp64 (some steps of its largest term, below 2^-40 here) and rounded once; the others are
    the same numbers."""
    got = f64(got)
    assert np.array_equal(np.isneginf(got), np.isneginf(want)) and np.array_equal(np.isnan(got), np.isnan(want))
    fine = np.isfinite(want)
    got, want = np.where(fine, got, 0), np.where(fine, want, 0)
    bad = np.abs(got - want) > 2.0 ** -24 * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -40
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def same(tc, dev, r, l, start, tokens, **kw):
    x = l.to(dev)
    out = torch.full(l.shape, float("nan"), device=dev)
    got = tc.logits_adjust(rules(r, dev), x, tensor(start, dev), tokens=None if tokens is None else tensor(tokens, dev), out=out)
    assert got is out
    want = logits_exact(f64(l), start, tokens, **r)
    close(got, want)
    return got, want


# one chunk, several, borders of words, chunks and lanes' four, odd ones
@pytest.mark.parametrize("xtype", ["F32", "F16", "BF16"])
@pytest.mark.parametrize("V", [1, 3, 31, 33, 1000, 1023, 1024, 1025, 4099, 32003, 70001])
def test_rules(tc, dev, V, xtype):
    rng = np.random.default_rng(V)
    same(tc, dev, *make(rng, V, [1, 4, 0, 9, 2], [50, 0, 7, 700, 1], bias=40, masks=3, xtype=xtype))


@pytest.mark.parametrize("leave", [("repetition",), ("frequency",), ("presence",), ("history", "history_start", "prompt"), ("prompt",),
                                   ("bias_start", "bias_token", "bias_value"), ("mask", "mask_of"), ("mask_of",),
                                   ("repetition", "frequency", "presence"), "all"])
@pytest.mark.parametrize("drafts", [True, False])
def test_left_out(tc, dev, leave, drafts):
    rng = np.random.default_rng(5)
    r, l, start, tokens = make(rng, 5003, [2, 3, 1], [30, 400, 0], bias=20, masks=6, drafts=drafts)
    r = {} if leave == "all" else {k: v for k, v in r.items() if k not in leave}
    got, want = same(tc, dev, r, l, start, tokens)
    if leave == "all":
        assert torch.equal(got.cpu(), l)


# (chunks: 2048 tokens, or 4096 where those of 2048 are more than two to a CU)
def test_many_sequences_and_chunk_sizes(tc, dev):
    """Chunks of 1024 to 8192 tokens of the vocabulary."""
    rng = np.random.default_rng(6)
    for V, S in ((9001, 2), (9001, 300), (20011, 300), (40009, 300)):
        same(tc, dev, *make(rng, V, [1] * S, list(rng.integers(0, 60, S)), bias=5, masks=4))


def test_long_history(tc, dev):
    """A history far longer than a workgroup, one token that comes most of the time."""
    rng = np.random.default_rng(7)
    r, l, start, tokens = make(rng, 3001, [3, 1], [100003, 20], bias=300)
    r["history"][:90000:2] = 17
    same(tc, dev, r, l, start, tokens)


# borders of the chunks of few sequences and of many
@pytest.mark.parametrize("V", [2047, 2048, 2049, 4095, 4096, 4097, 8193])
@pytest.mark.parametrize("n_seq", [3, 600])
def test_borders_of_chunks(tc, dev, V, n_seq):
    rng = np.random.default_rng(V + n_seq)
    rows, hist = ([int(n) for n in rng.integers(0, most, n_seq)] for most in (3, 20))
    same(tc, dev, *make(rng, V, rows, hist, bias=5, masks=2, xtype="BF16"))


# histories shorter than a load, and around what a workgroup loads at once, at the array's end and before it
@pytest.mark.parametrize("hist", [[0, 0], [1, 0], [0, 2], [1, 2], [3, 1], [2, 0], [2047, 1], [1, 2048], [2049, 0], [6143, 2], [3, 6144],
                                  [1, 6145], [10240, 3]])
def test_lengths_of_histories(tc, dev, hist):
    rng = np.random.default_rng(sum(hist))
    same(tc, dev, *make(rng, 300, [1, 2], hist))


def test_repeated_entries(tc, dev):
    """One token many times among the biases (added in their order: the sum depends on it), the history and the drafts."""
    V = 2000
    rng = np.random.default_rng(8)
    r, l, start, tokens = make(rng, V, [9], [64])
    tokens[:] = 77
    n = 500
    r.update(bias_start=np.array([0, n], np.int32), bias_token=np.full(n, 77, np.int32),
             bias_value=(rng.standard_normal(n) * 10.0 ** rng.integers(-4, 5, n)).astype(np.float32))
    r["bias_token"][::7] = 1999
    got, want = same(tc, dev, r, l, start, tokens)
    # the sum of a token's biases is the fp32 sum in the list's order
    back = np.float32(0)
    for v in r["bias_value"][r["bias_token"] == 1999]:
        back = np.float32(back + v)
    assert (r["history"] != 1999).all() and float(got[0, 1999]) == float(np.float32(float(l[0, 1999]) + float(back)))


def test_strange_numbers(tc, dev):
    """Tokens outside the vocabulary, lists whose borders lead outside, infinities and NaN among logits (masked: -infinity
    whatever they are), a row whose mask leaves nothing."""
    V = 1500
    rng = np.random.default_rng(9)
    r, l, start, tokens = make(rng, V, [2, 2, 1], [20, 20, 20], bias=10, masks=2)
    r["history"][:6] = [-1, V, 2 ** 31 - 1, -2 ** 31, V + 1000, 3]
    r["bias_token"][:2] = [V, -5]
    tokens[0], tokens[3] = -1, V
    l[0, :3] = torch.tensor([float("inf"), float("-inf"), float("nan")])
    l[1, 5] = float("nan")
    r["mask"][0] = 0
    r["mask"][1, 0] = -1 - (1 << 2) - (1 << 5)
    r["mask_of"][:] = [1, 1, 0, -1, 2 ** 31 - 1]
    got, want = same(tc, dev, r, l, start, tokens)
    assert torch.isneginf(got[2]).all() and not torch.isnan(got[0]).any() and float(got[0, 0]) == float("inf")
    # borders are held to the lists
    top = 2 ** 31 - 1
    r["history_start"][:] = [-5, 30, top, 10]
    r["bias_start"][:] = [-2 ** 31, 3, top, top]
    n, h = len(r["bias_token"]), 60
    inside = dict(r, history_start=None, bias_start=None)
    x = tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev), tokens=tensor(tokens, dev))
    # the same lists, each sequence with its own copy of what its borders leave
    hist = [r["history"][0:30], r["history"][30:h], r["history"][:0]]
    bias = [slice(0, min(3, n)), slice(min(3, n), n), slice(n, n)]
    inside.update(history=np.concatenate(hist), history_start=np.array([0, 30, h, h], np.int32),
                  bias_token=np.concatenate([r["bias_token"][b] for b in bias]),
                  bias_value=np.concatenate([r["bias_value"][b] for b in bias]),
                  bias_start=np.cumsum([0] + [b.stop - b.start for b in bias]).astype(np.int32))
    close(x, logits_exact(f64(l), start, tokens, **inside))


def test_rows_past_the_last_sequence(tc, dev):
    """A padded batch: its rows, and rows between borders that go backwards, stay as they are."""
    rng = np.random.default_rng(10)
    r, l, start, tokens = make(rng, 900, [2, 1, 3], [9, 9, 9])
    pad = torch.cat([l, l[:3]])
    out = torch.full(pad.shape, 7.0, device=dev)
    tc.logits_adjust(rules(r, dev), pad.to(dev), tensor(start, dev), tokens=tensor(np.concatenate([tokens, tokens[:3]]), dev), out=out)
    assert (out[6:] == 7.0).all()
    close(out[:6], logits_exact(f64(l), start, tokens, **r))
    out.fill_(7.0)
    tc.logits_adjust(rules(r, dev), pad.to(dev), tensor(np.array([0, 2, 1, 10 ** 6], np.int32), dev), out=out)
    assert torch.isfinite(out).all() and (out[0] != 7.0).any()


@pytest.mark.parametrize("xtype", ["F32", "BF16"])
def test_strides_and_in_place(tc, dev, xtype):
    rng = np.random.default_rng(11)
    r, l, start, tokens = make(rng, 1001, [2, 3], [90, 5], bias=9, masks=2, xtype=xtype)
    want, _ = same(tc, dev, r, l, start, tokens)
    for pad, at in ((3, 1), (24, 8)):
        wide = torch.full((5, 1001 + pad), 3.0, dtype=l.dtype, device=dev)
        to = torch.full((5, 1001 + pad), 7.0, device=dev)
        wide[:, at:at + 1001] = l.to(dev)
        tc.logits_adjust(rules(r, dev), wide[:, at:at + 1001], tensor(start, dev), tokens=tensor(tokens, dev), out=to[:, at:at + 1001])
        assert torch.equal(to[:, at:at + 1001], want)
        assert (to[:, :at] == 7.0).all() and (to[:, at + 1001:] == 7.0).all()
    if xtype == "F32":
        x = l.to(dev)
        assert tc.logits_adjust(rules(r, dev), x, tensor(start, dev), tokens=tensor(tokens, dev), out=x) is x
        assert torch.equal(x, want)
    for bad in (lambda: tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start[:2], dev)),
                lambda: tc.logits_adjust(rules(r, dev), l, tensor(start, dev)),
                lambda: tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev), tokens=tensor(tokens[:4], dev)),
                lambda: tc.logits_adjust(rules(r, dev), l.to(dev)[:, ::2], tensor(start, dev)),
                lambda: tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev), out=torch.zeros(5, 1001, device=dev).half())):
        with pytest.raises(tc_hip.TCError):
            bad()


def row_by_row(l, start, tokens, r):
    """logits_exact where prompt[s] below 0 counts -prompt[s] tokens of the history and of the step's behind it: every row by
    itself, with its tokens at the end of its history and what of all that was asked worked out here."""
    want = np.full(l.shape, np.nan)
    for s in range(len(start) - 1):
        had = r["history"][r["history_start"][s]:r["history_start"][s + 1]]
        for t in range(start[s], start[s + 1]):
            now = had if tokens is None else np.concatenate([had, tokens[start[s]:t + 1]])
            p = int(r["prompt"][s])
            one = dict(history=now, history_start=[0, len(now)], prompt=[-p if p < 0 else min(p, len(had))])
            one.update({n: r[n][s:s + 1] for n in ("repetition", "frequency", "presence")})
            if "bias_start" in r:
                one.update(bias_start=r["bias_start"][s:s + 2], bias_token=r["bias_token"], bias_value=r["bias_value"])
            if "mask" in r:
                one.update(mask=r["mask"], mask_of=r["mask_of"][t:t + 1])
            want[t] = logits_exact(l[t:t + 1], [0, 1], None, **one)[0]
    return want


# prompts from their first token on, chunks of prompts, prompts that end among the rows (drafts behind them), decoding
# sequences, and rows that several workgroups share
@pytest.mark.parametrize("xtype", ["F32", "BF16"])
@pytest.mark.parametrize("V", [50, 2049, 9001])
@pytest.mark.parametrize("rows,hist,asked", [
    ([30], [0], [30]), ([30], [0], [100]), ([9, 1, 5, 4], [0, 40, 20, 7], [9, 12, 24, 11]), ([6, 6], [3000, 10], [3003, 4]),
    ([1] * 300, [3] * 300, list(range(1, 301))), ([700], [20], [650]), ([2, 3], [5, 5], [2 ** 31, 2 ** 31 - 1])])
def test_tokens_that_were_asked(tc, dev, rows, hist, asked, V, xtype):
    """A prompt's own rows are asked, not answered: repetition alone counts them."""
    rng = np.random.default_rng(V + len(rows))
    r, l, start, tokens = make(rng, V, rows, hist, bias=3, masks=2, xtype=xtype)
    r["prompt"][:] = [-a for a in asked]
    x = tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev), tokens=tensor(tokens, dev))
    close(x, row_by_row(f64(l), start, tokens, r))
    # without the rows' tokens: of the history alone, as with the same number above 0
    x = tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev))
    r["prompt"][:] = [min(a, 2 ** 31 - 1) for a in asked]
    assert torch.equal(x, tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev)))
    # above 0: of the history alone, whatever else stands there
    got = tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev), tokens=tensor(tokens, dev))
    close(got, logits_exact(f64(l), start, tokens, **r))


def test_a_prompts_first_answer(tc, dev):
    """A prompt in chunks gets the logits that it gets as a history all at once, and no penalty on what it only asked."""
    rng = np.random.default_rng(12)
    V, n = 500, 37
    text = rng.integers(0, V, n).astype(np.int32)
    l = torch.from_numpy(rng.standard_normal((n, V)).astype(np.float32)).to(dev)
    f = lambda v: np.full(1, v, np.float32)  # noqa: E731
    base = dict(repetition=f(1.0), frequency=f(0.5), presence=f(0.7), prompt=np.array([-n], np.int32))
    for done in (0, 20, 36):
        r = dict(base, history=text[:done], history_start=np.array([0, done], np.int32))
        x = tc.logits_adjust(rules(r, dev), l[done:], tensor(np.array([0, n - done], np.int32), dev), tokens=tensor(text[done:], dev))
        assert torch.equal(x, l[done:])
    r = dict(base, history=text, history_start=np.array([0, n], np.int32))
    answer = np.array([text[3], text[3]], np.int32)
    x = tc.logits_adjust(rules(r, dev), l[:2], tensor(np.array([0, 2], np.int32), dev), tokens=tensor(answer, dev))
    close(x, logits_exact(f64(l[:2]), [0, 2], answer, **dict(r, prompt=[n])))
    assert (x != l[:2]).sum() == 2


def test_rows_of_no_sequence(tc, dev):
    """Rows in front of the first sequence, behind the last and between borders that go backwards stay as they are."""
    rng = np.random.default_rng(13)
    r, l, _, tokens = make(rng, 2100, [3, 3, 2], [9, 9, 9], bias=3, masks=2)
    for start, own in (([1, 3, 3, 5], [1, 2, 3, 4]), ([5, 2, 4, 4], [2, 3]), ([2, 4, 3, 3], [2, 3]), ([6, 6, 1, 0], [])):
        start = np.array(start, np.int32)
        out = torch.full(l.shape, 7.0, device=dev)
        tc.logits_adjust(rules(r, dev), l.to(dev), tensor(start, dev), tokens=tensor(tokens, dev), out=out)
        rest = [t for t in range(8) if t not in own]
        assert (out[rest] == 7.0).all(), start
        close(out[own], logits_exact(f64(l), start, tokens, **r)[own])
