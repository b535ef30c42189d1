"""The operators of a step together, as a serving program uses them: plan, norms, products of quantized weights, rotary
positions into the paged cache, attention, rules on logits, verification."""
import numpy as np
import pytest
import torch

import tc_hip
from paged import attn_bound, attn_exact
from qdata import Q8_0
from step import U, f64, logits_exact, norm_add_exact, plan_exact, rope_exact, tensor, turns_exact

pytestmark = pytest.mark.gpu

HID, HEADS, KV, D, FF, V, PAGE = 512, 8, 2, 64, 768, 1000, 16
EPS = float(np.float32(1e-6))


class Model:
    """Two blocks of random Q8_0 weights, with everything that a step keeps."""

    def __init__(self, tc, dev, n_seq, n_tokens, n_pages, seed=0, in_place=True):
        rng = np.random.default_rng(seed)
        self.tc, self.dev = tc, dev

        def weight(rows, cols):
            return tc.encode(Q8_0, tensor((rng.standard_normal((rows, cols)) / np.sqrt(cols)).astype(np.float32), dev)), rows, cols

        def norm(n):
            return tc_hip.Norm(tensor((1 + 0.2 * rng.standard_normal(n)).astype(np.float32), dev))

        self.blocks = [dict(qkv=weight((HEADS + 2 * KV) * D, HID), o=weight(HID, HEADS * D), up=weight(FF, HID), down=weight(HID, FF),
                            pre=norm(HID), mid=norm(HID), post=norm(HID), qn=norm(D), kn=norm(D),
                            cache=tc_hip.KVCache.empty(torch.float16, n_pages, KV, PAGE, D, device=dev)) for _ in range(2)]
        self.last, self.head = norm(HID), weight(V, HID)
        self.embed = tensor(rng.standard_normal((V, HID)).astype(np.float32), dev)
        self.rope = tc_hip.Rope(D, 1e4)
        z = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
        self.new, self.tokens = z(n_seq), z(n_tokens)
        free = z(3)
        free[1] = n_pages
        ring = torch.from_numpy(rng.permutation(n_pages).astype(np.int32)).to(dev)
        self.plan = tc_hip.KVPlan(self.new, z(n_seq), z(n_seq), z(n_seq, 8), ring, free, PAGE, n_tokens, in_place=in_place)
        self.history, self.history_start = z(n_seq * 128), torch.arange(0, 128 * n_seq + 1, 128, dtype=torch.int32, device=dev)
        self.history.fill_(-1)
        f = lambda v: torch.full((n_seq,), v, device=dev)  # noqa: E731
        mask = torch.full((2, (V + 31) // 32), -1, dtype=torch.int32, device=dev)
        mask[1, 3:9] = 0
        self.mask_of = torch.arange(n_tokens, dtype=torch.int32, device=dev) % 3 - 1
        self.rules = tc_hip.LogitRules(f(1.3), f(0.2), f(0.4), self.history, self.history_start, None,
                                       torch.arange(0, n_seq + 1, dtype=torch.int32, device=dev), z(n_seq) + 5, f(2.0), mask, self.mask_of)
        u = np.random.default_rng(seed + 1)
        self.accept_u, self.sample_u = (tensor(u.random(n).astype(np.float32), dev) for n in (n_tokens, n_seq))
        self.temperature = f(0.8)
        tc.attn_reserve(HEADS, n_tokens)
        tc._check(tc.lib.tc_gemv_reserve(FF, n_tokens))

    def product(self, w, x):
        return self.tc.gemv(Q8_0, w[0], x, w[1], w[2]) if x.shape[0] <= 8 else self.tc.gemm(Q8_0, w[0], x, w[1], w[2])

    def step(self, seen=None):
        """One step of the tokens in self.tokens; `seen` collects every operator's inputs and outputs."""
        tc, say = self.tc, (lambda *a: seen.append(a)) if seen is not None else (lambda *a: None)
        b = tc.kv_plan(self.plan).batch
        h = self.embed[self.tokens.long()]
        x = tc.norm(h, self.blocks[0]["pre"])
        say("norm", h, None, self.blocks[0]["pre"], None, None, x)
        for i, w in enumerate(self.blocks):
            qkv = self.product(w["qkv"], x).view(-1, HEADS + 2 * KV, D)
            q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:]
            r = tc.rope_kv_write(w["cache"], b, self.rope, q, k, v, q_norm=w["qn"].weight, k_norm=w["kn"].weight)
            say("rope", i, q, k, r)
            o = tc.attn(w["cache"], b, r, D ** -0.5)
            say("attn", i, r, o)
            y = self.product(w["o"], o.view(-1, HEADS * D))
            h2, x = tc.norm_add(h, y, pre=w["mid"])
            say("norm", h, y, w["mid"], None, h2, x)
            y = self.product(w["down"], torch.relu(self.product(w["up"], x)))
            nxt = self.blocks[i + 1]["pre"] if i == 0 else self.last
            h, x = tc.norm_add(h2, y, pre=nxt, post=w["post"], scale=0.5)
            say("norm", h2, y, nxt, w["post"], h, x)
        raw = self.product(self.head, x)
        out = tc.logits_adjust(self.rules, raw, self.plan.start, tokens=self.tokens)
        say("logits", raw, out)
        n, tok = tc.spec_verify(out, self.tokens, self.plan.start, self.temperature, self.accept_u, self.sample_u)
        return h, out, n, tok


def test_step_against_64_bits(tc, dev):
    """Prompts, drafted tokens, a sequence without tokens and one that ends, over four steps: each operator's outputs for
    the inputs it had, from its definition."""
    rng = np.random.default_rng(0)
    m = Model(tc, dev, 4, 40, 24)
    turns, _ = turns_exact(D, 1e4)
    p = m.plan
    for new in ([30, 5, 0, 3], [2, 9, 17, 1], [1, -1, 4, 8], [3, 20, 1, -1]):
        m.new.copy_(tensor(np.array(new, np.int32), dev))
        m.tokens.copy_(tensor(rng.integers(0, V, 40).astype(np.int32), dev))
        m.history.copy_(tensor(rng.integers(0, 60, 4 * 128).astype(np.int32), dev))
        state = [t.cpu().numpy().copy() for t in (p.held, p.pages, p.table, p.ring, p.free)]
        want = plan_exact(new, *state, PAGE, 40)
        assert want["free_out"][2] == 0
        seen = []
        _, out, n, tok = m.step(seen)
        for name in ("start", "length", "pages_out", "free_out", "position", "slot", "table", "ring"):
            assert np.array_equal(getattr(p, name).cpu().numpy(), want[name]), name
        T = int(want["start"][-1])
        pos = want["position"][:T]

        class Geometry:  # what paged.attn_exact asks of a batch
            kv_heads = KV

            def __init__(self, cache):
                self.cache = cache

            def value(self, name):
                return f64(getattr(self.cache, name))

            def rows(self):
                for t in range(T):
                    yield t, int(want["sequence"][t]), int(pos[t])

            def slot(self, s, j):
                return int(want["table"][s, j // PAGE]), j % PAGE

        for kind, *a in seen:
            if kind == "norm":
                h, y, pre, post, h2, x = a
                of = lambda q: None if q is None else (f64(q.weight), None, EPS, "rms", 0.0)  # noqa: E731
                e = norm_add_exact(f64(h), None if y is None else f64(y), of(pre), of(post), None, False, 0.5 if post else 1.0)
                for got, w, err in ((h2, e[0], e[1]), (x, e[2], e[3])):
                    # (rows past the last sequence hold whatever the memory of attention's output did)
                    assert got is None or (np.abs(f64(got) - w) <= err + U * (np.abs(w) + err))[:T].all()
            elif kind == "rope":
                i, q, k, r = a
                e, err = rope_exact(f64(q)[:T], pos, turns, D, "half", 1.0, f64(m.blocks[i]["qn"].weight), EPS)
                assert (np.abs(f64(r)[:T] - e) <= err + U * (np.abs(e) + err)).all()
                e, err = rope_exact(f64(k)[:T], pos, turns, D, "half", 1.0, f64(m.blocks[i]["kn"].weight), EPS)
                held = f64(m.blocks[i]["cache"].k).transpose(0, 2, 1, 3).reshape(-1, KV, D)[want["slot"][:T]]
                assert (np.abs(held - e) <= err + 2.0 ** -11 * (np.abs(e) + err) + 2.0 ** -25).all()
            elif kind == "attn":
                i, r, o = a
                e = attn_exact(Geometry(m.blocks[i]["cache"]), f64(r), D ** -0.5)
                bound = attn_bound("F32", "F16", D, 64, *e)
                assert (np.abs(f64(o) - e[0])[:T] <= bound[:T]).all()
            else:
                raw, got = a
                R = m.rules.held
                e = logits_exact(f64(raw)[:T], want["start"], m.tokens.cpu().numpy(), *[
                    t.cpu().numpy() for t in R[:3]], m.history.cpu().numpy(), m.history_start.cpu().numpy(), None,
                    np.arange(5), np.full(4, 5), np.full(4, 2.0, np.float32), R[-2].cpu().numpy(), m.mask_of.cpu().numpy())
                g = f64(got)[:T]
                assert np.array_equal(np.isfinite(g), np.isfinite(e))
                fine = np.isfinite(e)
                assert (np.abs(g[fine] - e[fine]) <= U * np.abs(e[fine]) * 1.001 + 2.0 ** -40).all()
                # a token that its mask forbids is never chosen
                first = want["start"][:4]
                for s in range(4):
                    if want["start"][s + 1] > first[s]:
                        row = first[s] + int(n[s])
                        assert int(tok[s]) >= 0 and np.isfinite(e[row, int(tok[s])])


def test_step_in_a_graph_and_on_another_stream(tc, dev):
    """The whole step captured once: replays, with eager work between them, walk through the sequences' lengths as the eager
    steps of a second model do on a stream of its own, bit for bit."""
    rng = np.random.default_rng(1)
    a, b = (Model(tc, dev, 3, 8, 20) for _ in range(2))
    side = torch.cuda.Stream()
    for m in (a, b):  # (sizes the scratch)
        m.step()
        for blk in m.blocks:
            blk["cache"].k.zero_()
            blk["cache"].v.zero_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = a.step()
    for step in range(6):
        new = rng.integers(0, 3, 3).astype(np.int32) if step != 4 else np.array([1, -1, 2], np.int32)
        tokens = rng.integers(0, V, 8).astype(np.int32)
        for m in (a, b):
            m.new.copy_(tensor(new, dev))
            m.tokens.copy_(tensor(tokens, dev))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = b.step()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        T = int(new.clip(0).sum())
        assert torch.equal(a.plan.length, b.plan.length) and torch.equal(a.plan.slot, b.plan.slot)
        for x, y in zip(got[:2], want[:2]):
            assert torch.equal(x[:T], y[:T]), step
        assert torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])


def test_calls_at_once(tc, dev):
    """None of the operators shares memory with another call: two streams at the same time give what one call gives."""
    rng = np.random.default_rng(2)
    h, y = (tensor(rng.standard_normal((512, 2048)).astype(np.float32), dev) for _ in range(2))
    n = tc_hip.Norm(torch.ones(2048, device=dev))
    x = tensor(rng.standard_normal((600, 8, 128)).astype(np.float32), dev)
    pos = tensor(np.arange(600, dtype=np.int32) * 37, dev)
    rope = tc_hip.Rope(128)
    l = tensor(rng.standard_normal((20, 30000)).astype(np.float32), dev)
    start = torch.arange(21, dtype=torch.int32, device=dev)
    rules = tc_hip.LogitRules(repetition=torch.full((20,), 1.2, device=dev), history=tensor(rng.integers(0, 30000, 4000).astype(np.int32), dev),
                              history_start=torch.arange(0, 4001, 200, dtype=torch.int32, device=dev))

    def work():
        return [*tc.norm_add(h, y, pre=n), tc.rope(rope, x, pos), tc.logits_adjust(rules, l, start)]

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
    torch.cuda.synchronize()
    for outs in got:
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_calls_without_rows(tc, dev):
    """Nothing to do is done anywhere."""
    z = lambda *n: torch.zeros(n, device=dev)  # noqa: E731
    i = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
    cache = tc_hip.KVCache.empty(torch.float16, 2, 2, 16, 64, device=dev)
    rope = tc_hip.Rope(64)
    for batch in (tc_hip.KVBatch(i(2), i(1), i(1, 2)), tc_hip.KVBatch(i(1), i(0), i(0, 2))):
        assert tc.rope_kv_write(cache, batch, rope, z(0, 4, 64), z(0, 2, 64), z(0, 2, 64)).shape == (0, 4, 64)
    q = z(3, 4, 64) + 5
    tc.rope_kv_write(cache, tc_hip.KVBatch(i(1), i(0), i(0, 2)), rope, q, z(3, 2, 64) + 1, z(3, 2, 64) + 1, out=q)
    assert (q == 5).all() and not cache.k.any() and not cache.v.any()
    assert tc.logits_adjust(tc_hip.LogitRules(), z(0, 100), i(1)).shape == (0, 100)
    l = z(2, 100) + 3
    assert tc.logits_adjust(tc_hip.LogitRules(), l, i(1), out=l) is l and (l == 3).all()
    h, x = tc.norm_add(z(0, 64), z(0, 64), pre=tc_hip.Norm())
    assert h.shape == x.shape == (0, 64)


def test_frequencies_are_there_when_made(tc, dev):
    """A rope made on one stream serves another at once."""
    x, pos = torch.ones(64, 1, 128, device=dev), torch.arange(64, dtype=torch.int32, device=dev)
    want = tc.rope(tc_hip.Rope(128, 1e6, scaling="yarn", factor=4.0, original=4096), x, pos)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        rope = tc_hip.Rope(128, 1e6, scaling="yarn", factor=4.0, original=4096)
        with torch.cuda.stream(side):
            got = tc.rope(rope, x, pos)
        side.synchronize()
        assert torch.equal(got, want)


def test_prompts_in_chunks_under_rules(tc, dev):
    """Plan and rules of a captured step, replayed while prompts come in chunks beside sequences that answer: a prompt's tokens
    are asked in whichever step they come, answers count from the first, and nothing of a step stays for the next."""
    rng = np.random.default_rng(3)
    S, T, room, vocab = 3, 16, 64, 300
    z = lambda *n: torch.zeros(n, dtype=torch.int32, device=dev)  # noqa: E731
    asked = np.array([25, 7, 1], np.int32)
    text = [list(rng.integers(0, 40, n)) for n in asked]
    new, tokens, history = z(S), z(T), z(S * room)
    free = tensor(np.array([0, 30, 0], np.int32), dev)
    plan = tc_hip.KVPlan(new, z(S), z(S), z(S, 8), torch.arange(30, dtype=torch.int32, device=dev), free, PAGE, T, in_place=True)
    r = dict(repetition=np.array([1.3, 1.0, 0.7], np.float32), frequency=np.array([0.2, 0.5, -0.3], np.float32),
             presence=np.array([0.4, 0.9, 0.1], np.float32))
    rules = tc_hip.LogitRules(**{k: tensor(v, dev) for k, v in r.items()}, history=history, history_start=z(S + 1),
                              prompt=tensor(-asked, dev))
    starts = rules.held[4]
    raw = tensor(rng.standard_normal((T, vocab)).astype(np.float32), dev)
    out = torch.full((T, vocab), 7.0, device=dev)

    def step():
        tc.kv_plan(plan)
        tc.logits_adjust(rules, raw, plan.start, tokens=tokens, out=out)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    done = [0, 0, 0]
    for chunk in ([12, 3, 1], [8, 4, 2], [5, 2, 0], [1, 1, 1], [2, 3, 1]):
        rows = []
        for s, n in enumerate(chunk):
            while len(text[s]) < done[s] + n:  # what it answers
                text[s].append(int(rng.integers(0, 40)))
            rows += text[s][done[s]:done[s] + n]
        past = [text[s][:done[s]] for s in range(S)]
        sums = np.concatenate([[0], np.cumsum([len(p) for p in past])]).astype(np.int32)
        new.copy_(tensor(np.array(chunk, np.int32), dev))
        tokens.copy_(tensor(np.array(rows + [5] * (T - len(rows)), np.int32), dev))
        flat = np.full(S * room, 7, np.int32)
        flat[:sums[-1]] = [t for p in past for t in p]
        history.copy_(tensor(flat, dev))
        starts.copy_(tensor(sums, dev))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        start = np.concatenate([[0], np.cumsum(chunk)])
        assert plan.start.tolist() == list(start) and int(plan.free_out[2]) == 0
        got = f64(out)
        assert (got[start[-1]:] == 7.0).all()
        for s in range(S):
            one = {k: v[s:s + 1] for k, v in r.items()}
            for t in range(start[s], start[s + 1]):
                now = np.array(text[s][:done[s] + t - start[s] + 1])
                e = logits_exact(f64(raw)[t:t + 1], [0, 1], None, history=now, history_start=[0, len(now)], prompt=asked[s:s + 1], **one)[0]
                assert (np.abs(got[t] - e) <= U * np.abs(e) * 1.001 + 2.0 ** -40).all(), (chunk, s, t)
            done[s] += chunk[s]


def test_frequencies_made_in_a_graph(tc, dev):
    """A rope made during a capture is filled by each replay, in front of the calls that use it."""
    x, pos = torch.ones(64, 1, 128, device=dev), torch.arange(64, dtype=torch.int32, device=dev)
    want = tc.rope(tc_hip.Rope(128, 1e6, scaling="linear", factor=4.0), x, pos)
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rope = tc_hip.Rope(128, 1e6, scaling="linear", factor=4.0)
        tc.rope(rope, x, pos, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert torch.equal(tc.rope(rope, x, pos), want)
