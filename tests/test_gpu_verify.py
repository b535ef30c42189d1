"""Verification of drafted tokens (tc_spec_verify) against its definition in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def pick(w, u):
    """The lowest token whose running sum passes u of all; the last of any weight if none."""
    cum = np.cumsum(w)
    past = np.nonzero(cum > u * cum[-1])[0]
    return int(past[0]) if len(past) else int(np.nonzero(w > 0)[0][-1])


def verify_exact(logits, tokens, start, temperature, accept_u, sample_u, probs):
    n_acc, nxt = [], []
    T, V = logits.shape
    for s in range(len(start) - 1):
        b, e = start[s], start[s + 1]
        if b == e:
            n_acc.append(0), nxt.append(-1)
            continue
        for i in range(e - b):
            row = logits[b + i].astype(np.float64)
            good = np.isfinite(row.max()) and not np.isnan(row).any()
            greedy = not temperature[s] > 0
            p = np.zeros(V)
            if good and greedy:
                p[int(row.argmax())] = 1
            elif good:
                p = np.exp((row - row.max()) / np.float64(temperature[s]))
                p /= p.sum()
            if i == e - b - 1:
                x, w = None, p
                break
            x = int(tokens[b + i + 1])
            inside = 0 <= x < V
            q = 1.0 if probs is None else float(probs[b + i, x]) if inside else 0.0
            take = good and inside and (p[x] == 1 if greedy else float(accept_u[b + i]) * q < p[x])
            if take:
                continue
            if probs is not None:
                w = np.fmax(p - probs[b + i].astype(np.float64), 0)
            else:
                w = p.copy()
                if inside:
                    w[x] = 0
            if greedy or not w.sum() > 0:
                w = p
            break
        n_acc.append(i)
        nxt.append(-1 if not good else int(row.argmax()) if greedy else pick(w, float(sample_u[s])))
    return np.array(n_acc, np.int32), np.array(nxt, np.int32)


def problem(seed, counts, V, probs, temps=None, pad=0):
    rng = np.random.default_rng(seed)
    start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    T, S = int(start[-1]) + pad, len(counts)
    logits = (2 * rng.standard_normal((T, V))).astype(np.float32)
    for t in range(T):
        logits[t, rng.integers(0, V, 3)] += 6
    d = logits + 0.7 * rng.standard_normal((T, V)).astype(np.float32)
    d = np.exp(d - d.max(1, keepdims=True))
    d = (d / d.sum(1, keepdims=True)).astype(np.float32)
    tokens = rng.integers(0, V, T).astype(np.int32)
    for t in range(1, T):
        if rng.random() < 0.7:
            tokens[t] = int(logits[t - 1].argmax()) if rng.random() < 0.5 else pick(d[t - 1].astype(np.float64), rng.random())
    temps = (0.4 + rng.random(S)).astype(np.float32) if temps is None else np.array(temps, np.float32)
    return [logits, tokens, start, temps, rng.random(T).astype(np.float32), rng.random(S).astype(np.float32),
            d if probs else None]


def check(tc, dev, p):
    t = [None if a is None else torch.from_numpy(a).to(dev) for a in p]
    got = tc.spec_verify(*t[:6], draft_probs=t[6])
    want = verify_exact(*p)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w), (g, w)
    return want


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("V", [1, 2, 5, 63, 1000, 4097, 32001, 152064])
def test_verify_vocabularies(tc, dev, V, probs):
    check(tc, dev, problem(V, [5, 1, 3, 9], V, probs))


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("counts", [[1], [9], [0, 3, 0], [2] * 70, [1] * 200, [40, 1], [300], [8] * 129])
def test_verify_batches(tc, dev, counts, probs):
    """One sequence, many, empty ones, long chunks; rows past the last sequence are no one's."""
    n, _ = check(tc, dev, problem(len(counts), counts, 777, probs, pad=2))
    if counts == [2] * 70:
        assert n.min() == 0 and n.max() == 1  # (seeded: drafts are taken and rejected)


@pytest.mark.parametrize("probs", [False, True])
def test_verify_many_sequences(tc, dev, probs):
    """Thousands of sequences, most of them of no row, one or two."""
    check(tc, dev, problem(17, [1, 0, 2, 0, 0, 5] * 800, 37, probs, pad=3))


@pytest.mark.parametrize("probs", [False, True])
def test_verify_greedy_and_mixed(tc, dev, probs):
    """Temperature 0, with ties (the lowest token), beside sampled sequences."""
    p = problem(3, [5] * 40, 5000, probs, temps=[0.0, 0.7] * 20)
    p[0][::3, 4000] = p[0][::3].max(1)
    p[1][1::3] = p[0][0:-1:3].argmax(1)[:len(p[1][1::3])]
    n, _ = check(tc, dev, p)
    assert n.max() > 0


def test_verify_random_numbers_at_the_ends(tc, dev):
    """0 takes the first token of any weight, a number next to 1 the last; a draft of probability 0 is taken
    by 0 only where its draft probability is 0 too and its own is not."""
    p = problem(4, [2] * 64, 300, True)
    p[4][:32] = 0.0
    p[4][32:64] = np.float32(1 - 2 ** -24)
    p[5][::2] = 0.0
    p[5][1::2] = np.float32(1 - 2 ** -24)
    p[0][:, :7] = -np.inf
    p[0][:, -9:] = -np.inf
    p[6][:, 50] = 0
    p[1][1:20] = 50
    p[1][20:40] = 3
    check(tc, dev, p)


def test_verify_same_distribution(tc, dev):
    """A draft model that is the target: nothing is left where it is rejected, so p itself is drawn from."""
    p = problem(5, [4] * 30, 64, True, temps=[1.0] * 30)
    p[0][:] = 0.0  # 1/64 each, exactly, on both sides
    p[6][:] = 1 / 64
    p[4][:] = 1.0  # (no draft is taken)
    n, _ = check(tc, dev, p)
    assert n.max() == 0


@pytest.mark.parametrize("probs", [False, True])
def test_verify_odd_values(tc, dev, probs):
    """Drafts outside the vocabulary, masked tokens, NaN and infinite logits."""
    p = problem(6, [3] * 12, 2000, probs, temps=[0.8, 0.0] * 6)
    p[1][1], p[1][4], p[1][7] = -1, 2000, 2 ** 31 - 1
    p[0][9, :] = -np.inf
    p[0][12, 77] = np.nan
    p[0][15, 1999] = np.nan
    p[0][18, 5] = np.inf
    p[0][21, 10:] = -np.inf
    p[0][24, 100:1900] = -np.inf
    p[0][27, 3] = 3e38
    check(tc, dev, p)


def test_verify_flat_distribution(tc, dev):
    """A vocabulary whose tokens are all alike: a random number's token is its product with the size."""
    V, S = 152064, 64
    start = np.arange(S + 1, dtype=np.int32)
    u = np.random.default_rng(7).random(S).astype(np.float32)
    p = [np.zeros((S, V), np.float32), np.zeros(S, np.int32), start, np.ones(S, np.float32), u, u, None]
    t = [None if a is None else torch.from_numpy(a).to(dev) for a in p]
    _, tok = tc.spec_verify(*t[:6])
    assert np.array_equal(tok.cpu().numpy(), np.floor(u.astype(np.float64) * V).astype(np.int32))


def test_verify_as_a_graph(tc, dev):
    p = problem(8, [3, 6, 1, 9, 0, 5], 3001, True)
    q = problem(9, [9, 1, 2, 5, 4, 3], 3001, True)
    live = [torch.from_numpy(a).to(dev) for a in p]
    tc.attn_reserve(1, 24)
    tc.spec_verify(*live[:6], draft_probs=live[6])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = tc.spec_verify(*live[:6], draft_probs=live[6])
    for turn in range(4):
        now = (p, q)[turn % 2]
        for a, b in zip(live, now):
            a.copy_(torch.from_numpy(b))
        for o in out:
            o.fill_(-7)
        check(tc, dev, problem(turn, [2] * 100, 900, False))  # eager work of another size
        g.replay()
        torch.cuda.synchronize()
        for o, w in zip(out, verify_exact(*now)):
            assert np.array_equal(o.cpu().numpy(), w), turn


def test_draft_step(tc, dev):
    """A chunk of drafted tokens through the operators as a serving step has them: keys and values written,
    attention over the cache, logits from the rows through the quantized LM head, verification; rejected
    tokens' slots are written over by the next step."""
    import tc_hip
    rng = np.random.default_rng(11)
    H, KV, D, V = 8, 2, 64, 2048
    hid = H * D
    g = torch.Generator().manual_seed(1)
    head = tc.encode(tc_hip.Q8_0, (torch.randn(V, hid, generator=g) * 0.5).to(dev))
    wk = tc.encode(tc_hip.Q4_K, torch.randn(KV * D, hid, generator=g).to(dev))
    emb = torch.randn(V, hid, generator=g).to(dev)
    cache = tc_hip.KVCache.empty(torch.int8, 12, KV, 16, D, device=dev)
    table = torch.arange(12, dtype=torch.int32).reshape(2, 6).flip(1).contiguous().to(dev)

    def step(tokens, lengths):
        """Logits of a chunk of 4 tokens of each of two sequences."""
        start = torch.tensor([0, 4, 8], dtype=torch.int32, device=dev)
        x = emb[tokens.long()]
        kv = tc.gemv(tc_hip.Q4_K, wk, x, KV * D, hid).reshape(8, KV, D)
        batch = tc_hip.KVBatch(start, lengths, table)
        tc.kv_write(cache, batch, kv, kv)
        o = tc.attn(cache, batch, x.reshape(8, H, D), D ** -0.5)
        return start, tc.gemv(tc_hip.Q8_0, head, o.reshape(8, hid), V, hid), kv

    lengths = torch.tensor([4, 4], dtype=torch.int32, device=dev)
    tokens = torch.from_numpy(rng.integers(0, V, 8).astype(np.int32)).to(dev)
    kept = [[], []]  # the keys of the tokens that stay
    u = lambda n: torch.rand(n, generator=g).to(dev)  # noqa: E731
    for turn in range(6):
        start, logits, kv = step(tokens, lengths)
        args = (logits, tokens, start, torch.full((2,), 40.0, device=dev), u(8) * 1e-3, u(2))
        n, nxt = tc.spec_verify(*args)
        want = verify_exact(*(a.cpu().numpy() for a in args), None)
        assert np.array_equal(n.cpu().numpy(), want[0]) and np.array_equal(nxt.cpu().numpy(), want[1])
        for s in range(2):
            kept[s] += [kv[4 * s + i] for i in range(1 + int(n[s]))]
        lengths = lengths + n + 1
        lengths = lengths.to(torch.int32)
        tokens = torch.from_numpy(rng.integers(0, V, 8).astype(np.int32)).to(dev)
        tokens[0], tokens[4] = nxt[0], nxt[1]
        # the chunk just written may reach past the kept tokens, never over them
        at = torch.tensor([len(k) for k in kept], dtype=torch.int32, device=dev)
        whole = tc_hip.KVBatch(torch.cat([at.new_zeros(1), at.cumsum(0).to(torch.int32)]), at, table)
        back, _ = tc.kv_read(cache, whole, int(at.sum()), torch.float32)
        rows = torch.stack(kept[0] + kept[1])
        assert ((back - rows).abs() <= rows.abs().amax(-1, keepdim=True) / 127 * 0.5001).all()
        if int(lengths.max()) > 90:
            break


def verify_into(tc, dev, p):
    """The C entry into outputs that hold no token yet."""
    t = [None if a is None else torch.from_numpy(a).to(dev) for a in p]
    logits, tokens, start, temperature, accept_u, sample_u, probs = t
    out = [torch.full((len(p[2]) - 1,), -7, dtype=torch.int32, device=dev) for _ in range(2)]
    ptr = [x.data_ptr() if x is not None else None for x in (logits, probs)]
    rc = tc.lib.tc_spec_verify(*ptr, logits.shape[1], len(p[2]) - 1, logits.shape[0],
                               *(x.data_ptr() for x in (start, tokens, temperature, accept_u, sample_u, *out)), tc._stream())
    assert rc == 0, tc.lib.tc_last_error()
    return [o.cpu().numpy() for o in out]


def draws(logits, u):
    """One row of each sequence, nothing drafted."""
    S = len(u)
    return [logits, np.zeros(S, np.int32), np.arange(S + 1, dtype=np.int32), np.ones(S, np.float32), np.zeros(S, np.float32),
            np.asarray(u, np.float32), None]


def equal_tokens(where, u):
    """For each random number the tokens it may draw among equal ones: the lowest whose share of the sum up to it
    exceeds u, and where u is a border, which a rounding of that sum moves to either side, the one before it too."""
    n = len(where)
    for x in u:
        k = int(np.floor(float(x) * n))
        yield {int(where[k])} | ({int(where[k - 1])} if k and float(x) * n == k else set())


@pytest.mark.parametrize("n", [10, 12, 14, 20, 40, 96])
def test_verify_draws_on_borders_of_few(tc, dev, n):
    """A few equal tokens of a vocabulary, anywhere: random numbers on the borders between them, each draws a token."""
    V, u = 32768, np.arange(64) / 64
    rng = np.random.default_rng(n)
    for where in [np.arange(n) * (V // n), 512 * np.arange(n) % V + np.arange(n) // 64] + [rng.choice(V, n, False) for _ in range(6)]:
        where = np.sort(where)
        logits = np.full((64, V), -np.inf, np.float32)
        logits[:, where] = 1.25
        _, got = verify_into(tc, dev, draws(logits, u))
        for j, may in enumerate(equal_tokens(where, u)):
            assert got[j] in may, (j, got[j], may)
        for j in (16, 32, 48):  # alone: other slices
            _, one = verify_into(tc, dev, draws(logits[:1], u[j:j + 1]))
            assert one[0] in list(equal_tokens(where, u[j:j + 1]))[0], j


@pytest.mark.parametrize("V,S", [(128000, 48), (256000, 48), (50304, 64), (152064, 64), (1000, 1)])
def test_verify_draws_on_borders_of_flat_rows(tc, dev, V, S):
    """Vocabularies whose tokens are all alike, random numbers on a grid of 1/64."""
    where = np.arange(V)
    for first in range(0, 64, S):
        u = (first + np.arange(S)) % 64 / 64
        _, got = verify_into(tc, dev, draws(np.zeros((S, V), np.float32), u))
        for j, may in enumerate(equal_tokens(where, u)):
            # (sums of V roundings: a token further at most)
            assert got[j] in may or abs(got[j] - u[j] * V) <= 1, (u[j], got[j], may)


def test_verify_random_numbers_past_the_ends(tc, dev):
    """Numbers below 0 draw the first token of any weight; 1, more, and NaN the last one."""
    logits = np.full((7, 5000), -np.inf, np.float32)
    logits[:, [70, 900, 901, 4321]] = [0.5, -3, 2, 1]
    _, got = verify_into(tc, dev, draws(logits, [-1e-30, -0.5, -np.inf, 1, 1.5, np.inf, np.nan]))
    assert got.tolist() == [70, 70, 70, 4321, 4321, 4321, 4321]


@pytest.mark.parametrize("probs", [False, True])
def test_verify_temperature_without_end(tc, dev, probs):
    """An infinite temperature makes all tokens that are not masked alike, for drafts and draws."""
    p = problem(12, [4] * 20, 1000, probs, temps=[np.inf, 0.9] * 10)
    p[0][:, 200:300] = -np.inf
    p[0][::3, 700] = 3e38
    p[4][:] *= 2e-3
    flat = [a if a is None else a.copy() for a in p]
    for s in range(0, 20, 2):
        rows = flat[0][flat[2][s]:flat[2][s + 1]]
        rows[np.isfinite(rows)] = 0  # at temperature 1 the same
        flat[3][s] = 1
    got, want = verify_into(tc, dev, p), verify_exact(*flat)
    assert want[0][::2].max() > 0  # (seeded: some drafts are taken)
    for g, w in zip(got, want):
        assert np.array_equal(g, w), (g, w)


def test_verify_temperature_below_zero(tc, dev):
    """Negative temperatures and NaN are taken for 0."""
    p = problem(13, [3] * 8, 500, True, temps=[0.0, -0.0, -1.0, -np.inf, np.nan, -1e-45, 0.0, -0.7])
    zero = [a if a is None else a.copy() for a in p]
    zero[3][:] = 0
    for g, w in zip(verify_into(tc, dev, p), verify_exact(*zero)):
        assert np.array_equal(g, w), (g, w)
