"""tc_kv_plan: every number it writes against the same worked out by hand (tests/step.py)."""
import ctypes

import numpy as np
import pytest
import torch

import tc_hip
from step import plan_exact, tensor

pytestmark = pytest.mark.gpu

OUT = ("start", "length", "pages_out", "free_out", "sequence", "position", "slot", "table", "ring")


def state(rng, held, extra=(), width=None, ring=None, at=0, page=16):
    """Pages for sequences that hold `held` tokens (and extra[s] more), in a random order; the rest free."""
    n = [-(-h // page) + (extra[s] if s < len(extra) else 0) for s, h in enumerate(held)]
    R, W = ring or sum(n) + 40, width or max(n + [1]) + 8
    order = rng.permutation(R).astype(np.int32)
    table = np.full((len(held), W), -7, np.int32)  # entries that are not to be followed
    i = 0
    for s, k in enumerate(n):
        table[s, :k] = order[i:i + k]
        i += k
    r = np.full(R, -9, np.int32)
    for j in range(R - i):
        r[(at + j) % R] = order[i + j]
    return dict(held=np.array(held, np.int32), pages=np.array(n, np.int32), table=table, ring=r,
                free=np.array([at, R - i, 5], np.int32))


def run(tc, dev, st, new, page, n_tokens, in_place=False):
    t = {k: tensor(v, dev) for k, v in st.items()}
    p = tc_hip.KVPlan(tensor(np.array(new, np.int32), dev), t["held"], t["pages"], t["table"], t["ring"], t["free"], page,
                      n_tokens, in_place=in_place)
    return tc.kv_plan(p)


def check(p, want):
    for name in OUT:
        got = getattr(p, name).cpu().numpy()
        assert np.array_equal(got, want[name]), (name, np.argwhere(got != want[name])[:5], got, want[name])


def same(tc, dev, st, new, page, n_tokens, in_place=False):
    want = plan_exact(new, st["held"], st["pages"], st["table"], st["ring"], st["free"], page, n_tokens)
    check(run(tc, dev, st, new, page, n_tokens, in_place), want)
    return want


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("page", [1, 16, 48, 64])
@pytest.mark.parametrize("new", [[1], [1, 1, 1, 1, 1], [3, 0, 200, 1, 17], [0, 0, 0, 0, 0], [-1, 2, -1, 64, 0], [-1, -1, -1, -1, -1]])
def test_plan(tc, dev, new, page, in_place):
    rng = np.random.default_rng(page + len(new))
    held = [int(h) for h in rng.choice([0, 1, 15, 16, 17, 63, 64, 100], len(new))]
    st = state(rng, held, extra=[0, 2, 1, 0, 3], ring=600, at=590, page=page, width=320)
    want = same(tc, dev, st, new, page, sum(max(n, 0) for n in new) + 3, in_place)
    assert want["free_out"][2] == 0


@pytest.mark.parametrize("n_seq,most", [(1023, 3), (1024, 9), (1025, 40), (2500, 9), (300, 300)])
def test_plan_many(tc, dev, n_seq, most):
    """More sequences than threads, rows for a launch of their own, one ended in ten."""
    rng = np.random.default_rng(n_seq)
    held = [int(h) for h in rng.integers(0, 70, n_seq)]
    new = rng.integers(0, most + 1, n_seq).astype(np.int32)
    new[rng.random(n_seq) < 0.1] = -1
    st = state(rng, held, extra=list(rng.integers(0, 2, n_seq)), ring=n_seq * 40, at=n_seq * 40 - 3, width=40)
    same(tc, dev, st, new, 16, int(np.maximum(new, 0).sum()) + 70)


def test_plan_long_prompts(tc, dev):
    rng = np.random.default_rng(3)
    st = state(rng, [0, 100, 31, 5000], ring=3000, width=1100)
    same(tc, dev, st, [16000, 1, 4097, 9], 16, 16000 + 1 + 4097 + 9)
    same(tc, dev, st, [4094, 1, 0, 1], 16, 4096)  # the most rows that one workgroup looks up, and one more
    same(tc, dev, st, [4095, 1, 0, 1], 16, 4097)


def test_plan_shortage(tc, dev):
    """Too few pages: in the sequences' order, -1 in the table, counted, slots of -1; a page given back serves."""
    rng = np.random.default_rng(4)
    st = state(rng, [10, 20, 30, 40], ring=12, at=11)
    left = int(st["free"][1])
    want = same(tc, dev, st, [30, 40, 50, 60], 16, 180)
    assert want["free_out"][2] > 0 and (want["slot"] == -1).any()
    want = same(tc, dev, st, [30, 40, -1, 60], 16, 180)
    assert want["free_out"][2] < 10 - left
    # the next step takes up where this one was short
    nxt = dict(held=want["length"], pages=want["pages_out"], table=want["table"], ring=want["ring"], free=want["free_out"])
    same(tc, dev, nxt, [0, -1, 0, 1], 16, 3)


def test_plan_narrow_table(tc, dev):
    """More pages than the table has entries for: counted, not written, rows without a slot."""
    rng = np.random.default_rng(5)
    st = state(rng, [10, 20], ring=30, width=3)
    want = same(tc, dev, st, [100, 5], 16, 110)
    assert want["free_out"][2] == 4 and want["table"].shape == (2, 3)


def test_plan_cut_rows(tc, dev):
    """Fewer rows than the sequences bring: the last of them get fewer or none, and no longer for it."""
    rng = np.random.default_rng(6)
    st = state(rng, [10, 20, 0, 5])
    for n in (0, 1, 30, 31, 49):
        want = same(tc, dev, st, [30, 1, 18, 3], 16, n)
        assert want["start"][-1] == n
    same(tc, dev, st, [2 ** 31 - 1, 2 ** 31 - 1, 3, 4], 16, 50)


def test_plan_bad_numbers(tc, dev):
    """Arrays that hold anything at all lead nowhere outside."""
    rng = np.random.default_rng(7)
    st = state(rng, [10, 20, 30, 40, 50, 60], ring=64, width=6)
    top, low = 2 ** 31 - 1, -2 ** 31
    for held, pages, free, new in (
            ([low, -1, top, 2 ** 31 - 65, 2 ** 31 - 66, 0], [0, -3, top, low, 7, 6], [top, top, 0], [5, 0, 7, 9, 2, 3]),
            ([10, 20, 30, 40, 50, 60], [top, 1, 2, 3, 4, 5], [-5, 3, 0], [-1, low, 1, top, -1, 1]),
            ([10, 20, 30, 40, 50, 60], [6, 6, 6, 6, 6, 6], [63, 60, 0], [-1, -1, -1, -1, -1, 40]),  # (a ring without room)
            ([10, 20, 30, 40, 50, 60], [1, 2, 2, 3, 4, 4], [3, -1, 0], [16, 16, 16, 16, 16, 16])):
        bad = dict(st, held=np.array(held, np.int32), pages=np.array(pages, np.int32), free=np.array(free, np.int32))
        want = plan_exact(new, bad["held"], bad["pages"], bad["table"], bad["ring"], bad["free"], 16, 40)
        # (a length held to the largest leaves its first rows no position)
        want["position"] = np.where(want["position"] < 0, -1, want["position"])
        check(run(tc, dev, bad, new, 16, 40), want)


def test_plan_without_maps_or_sequences(tc, dev):
    """The rows' arrays may be left out; no sequences: no rows."""
    rng = np.random.default_rng(8)
    st = state(rng, [10, 20])
    p = run(tc, dev, st, [3, 30], 16, 40)
    for keep in ("sequence", "position", "slot", None):
        for n in ("start", "sequence", "position", "slot"):
            getattr(p, n).fill_(77)
        c = tc_hip._CPlan.from_buffer_copy(p.c)
        for n in ("sequence", "position", "slot"):
            if n != keep:
                setattr(c, n, None)
        assert tc.lib.tc_kv_plan(ctypes.byref(c), tc._stream()) == tc_hip.TC_OK
        want = plan_exact([3, 30], st["held"], st["pages"], st["table"], st["ring"], st["free"], 16, 40)
        assert p.start.tolist() == list(want["start"])
        for n in ("sequence", "position", "slot"):
            got = getattr(p, n).cpu().numpy()
            assert np.array_equal(got, want[n]) if n == keep else (got == 77).all()
    empty = dict(held=np.zeros(0, np.int32), pages=np.zeros(0, np.int32), table=np.zeros((0, 4), np.int32), ring=st["ring"],
                 free=st["free"])
    p = run(tc, dev, empty, [], 16, 5)
    assert p.start.tolist() == [0] and p.slot.tolist() == [-1] * 5 and p.free_out.tolist() == [0, int(st["free"][1]), 0]


def test_plan_steps_in_a_graph(tc, dev):
    """A captured step, replayed: lengths grow, pages come and go in place, as worked out by hand."""
    rng = np.random.default_rng(9)
    st = state(rng, [10, 0, 30, 64], ring=40, at=33, width=12)
    t = {k: tensor(v, dev) for k, v in st.items()}
    new = tensor(np.array([1, 1, 1, 1], np.int32), dev)
    p = tc_hip.KVPlan(new, t["held"], t["pages"], t["table"], t["ring"], t["free"], 16, 12, in_place=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tc.kv_plan(p)
    for step in range(12):
        n = rng.integers(0, 4, 4).astype(np.int32)
        n[rng.random(4) < 0.15] = -1
        new.copy_(tensor(n, dev))
        want = plan_exact(n, st["held"], st["pages"], st["table"], st["ring"], st["free"], 16, 12)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(p, want)
        st = dict(held=want["length"], pages=want["pages_out"], table=want["table"], ring=want["ring"], free=want["free_out"])


def test_plan_pages_in_two_tables(tc, dev):
    """Sequences with a common beginning: a sequence that ends gives back the first `pages` entries of its row. With its own
    pages moved there and `pages` their number, the common ones stay with the other sequence, and no page comes twice."""
    rng = np.random.default_rng(10)
    page, common = 16, 3
    st = state(rng, [70, 0, 40], ring=30, width=12)
    pages, table = st["pages"], st["table"]
    # the second sequence begins with the first one's first three pages, and has 20 tokens of its own behind them
    own = st["ring"][:2].copy()
    table[1, :common], table[1, common:common + 2] = table[0, :common], own
    pages[1], st["held"][1] = common + 2, common * page + 20
    st["free"][0], st["free"][1] = 2, st["free"][1] - 2
    want = same(tc, dev, st, [1, 30, 1], page, 40)
    st = dict(held=want["length"], pages=want["pages_out"], table=want["table"], ring=want["ring"], free=want["free_out"])
    mine = int(st["pages"][1]) - common
    assert mine == 4
    st["table"][1, :mine] = st["table"][1, common:common + mine].copy()
    st["pages"][1] = mine
    want = same(tc, dev, st, [1, -1, 1], page, 2)
    at, left = want["free_out"][:2]
    free = [int(want["ring"][(at + i) % 30]) for i in range(left)]
    used = [int(p) for s in (0, 2) for p in want["table"][s, :want["pages_out"][s]]]
    assert sorted(free + used) == list(range(30)) and want["free_out"][2] == 0
