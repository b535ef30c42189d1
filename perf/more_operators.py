"""The operators around a serving step's products and attention, as cases to time and compare.

A case is a dict of plain values; `op` names the operator:

  plan    rows, positions, cache slots and new pages of a step from its sequences' lengths (tc_kv_plan)
  rope    rotary positions of queries and keys, keys and values into the paged cache (tc_rope_kv_write)
  norm    residual stream + gated, normalised output of a block, and the next block's norm (tc_norm_add)
  logits  penalties for repeated tokens, biases and masks on logits (tc_logits_adjust)

Sequences' lengths come from a case's own numbers (`mix` seeds the choice), so that they do not change with the seed;
values, pages, tokens and random numbers do.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
X = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
C = {"F16": torch.float16, "BF16": torch.bfloat16, "E4M3": torch.float8_e4m3fn}


def listed():
    return [
        # A decode step of a few sequences: one token each. The smallest call, all latency.
        {"name": "plan_decode", "op": "plan", "n_seq": 16, "new_min": 1, "new_max": 1, "ctx_min": 100, "ctx_max": 16000,
         "mix": 0, "page": 16, "ended": 1},
        # A step of a busy server: chunks of prompts among decoding sequences, some that ended give their pages back.
        {"name": "plan_mixed", "op": "plan", "n_seq": 301, "new_min": 1, "new_max": 4096, "ctx_min": 0, "ctx_max": 16000,
         "mix": 1, "page": 64, "ended": 20},
        # One token of one sequence, fp32 rows as the decode products give them.
        {"name": "rope_1tok", "op": "rope", "x": "F32", "c": "F16", "n_seq": 1, "new_min": 1, "new_max": 1,
         "ctx_min": 1000, "ctx_max": 1000, "mix": 0, "heads": 28, "kv_heads": 4, "dim": 128, "page": 16, "n_rot": 128,
         "layout": "half", "scaling": "none", "norm": False},
        # Drafted tokens of a batch at far positions, heads normalised, an 8-bit cache, frequencies stretched.
        {"name": "rope_drafts", "op": "rope", "x": "BF16", "c": "E4M3", "n_seq": 64, "new_min": 1, "new_max": 8,
         "ctx_min": 500, "ctx_max": 120000, "mix": 2, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "n_rot": 128,
         "layout": "half", "scaling": "yarn", "norm": True},
        # A chunk of a long prompt; neighbouring dims are pairs, and half of a head is rotated.
        {"name": "rope_chunk", "op": "rope", "x": "BF16", "c": "BF16", "n_seq": 1, "new_min": 8190, "new_max": 8190,
         "ctx_min": 100001, "ctx_max": 100001, "mix": 0, "heads": 28, "kv_heads": 4, "dim": 128, "page": 64, "n_rot": 64,
         "layout": "pairs", "scaling": "bands", "norm": False},
        # Between two blocks of a decode step: the residual sum and the next norm.
        {"name": "norm_1tok", "op": "norm", "x": "F32", "h": "F32", "o": "F32", "rows": 1, "cols": 3584, "kind": "rms",
         "post": False, "gate": "none", "sigmoid": False, "scale": 1.0},
        # A decode batch: layer norms with biases, a gate for each channel.
        {"name": "norm_batch", "op": "norm", "x": "F32", "h": "F32", "o": "BF16", "rows": 64, "cols": 5120,
         "kind": "layer", "post": False, "gate": "channel", "sigmoid": False, "scale": 0.5},
        # A long prompt: norms behind and before the blocks, a gate for each token, 16-bit rows.
        {"name": "norm_prompt", "op": "norm", "x": "BF16", "h": "BF16", "o": "BF16", "rows": 8192, "cols": 5120,
         "kind": "rms", "post": True, "gate": "row", "sigmoid": True, "scale": 0.22},
        # Wide rows of an odd width, a gate for each value.
        {"name": "norm_wide", "op": "norm", "x": "F16", "h": "F32", "o": "F16", "rows": 1000, "cols": 17407,
         "kind": "rms", "post": False, "gate": "full", "sigmoid": True, "scale": 1.0},
        # One sequence's next token behind a chat of ordinary length.
        {"name": "logits_1seq", "op": "logits", "x": "F32", "n_seq": 1, "drafts_min": 0, "drafts_max": 0, "mix": 0,
         "vocab": 152064, "hist_min": 2000, "hist_max": 2000, "bias": 20, "mask": False},
        # Drafted tokens of a batch with long histories, under grammars that differ from row to row.
        {"name": "logits_drafts", "op": "logits", "x": "F32", "n_seq": 48, "drafts_min": 0, "drafts_max": 8, "mix": 3,
         "vocab": 152064, "hist_min": 100, "hist_max": 32000, "bias": 300, "mask": True},
        # A large decode batch, 16-bit logits of an odd vocabulary.
        {"name": "logits_batch", "op": "logits", "x": "BF16", "n_seq": 256, "drafts_min": 0, "drafts_max": 0, "mix": 4,
         "vocab": 32003, "hist_min": 10, "hist_max": 4000, "bias": 8, "mask": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "rope", "norm", "norm", "logits", "logits"])
    mix = rng.randrange(1 << 30)
    if op == "plan":
        n_seq = _log(rng, 1, 500)
        hi = rng.choice([1, 1, 9, _log(rng, 2, 4096)])
        return {"op": op, "n_seq": n_seq, "new_min": rng.choice([0, 1]), "new_max": hi, "ctx_min": 0,
                "ctx_max": _log(rng, 10, 30000), "mix": mix, "page": rng.choice([16, 16, 32, 48, 64, 128, 256]),
                "ended": rng.choice([0, 1, n_seq // 10])}
    if op == "rope":
        dim, kv = rng.choice([64, 80, 96, 128, 128, 128, 192, 256]), rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 7])
        n_seq = _log(rng, 1, 64)
        most = 8190 * 36 * 128 // (n_seq * (heads + 2 * kv) * dim)
        hi = max(1, min(rng.choice([1, 8, _log(rng, 1, 8190)]), most))
        return {"op": op, "x": rng.choice(sorted(X)), "c": rng.choice(sorted(C)), "n_seq": n_seq,
                "new_min": max(1, hi // rng.choice([1, 3, 50])), "new_max": hi, "ctx_min": 0,
                "ctx_max": max(1, min(_log(rng, 1, 130000), 40_000_000 // (n_seq * kv * dim // 64))), "mix": mix,
                "heads": heads, "kv_heads": kv, "dim": dim, "page": rng.choice([16, 32, 48, 64, 128]),
                "n_rot": rng.choice([dim, dim, dim // 2, dim // 4, dim - 6]), "layout": rng.choice(["half", "pairs"]),
                "scaling": rng.choice(["none", "linear", "ntk", "yarn", "bands"]), "norm": rng.random() < 0.4}
    if op == "norm":
        cols = rng.choice([_log(rng, 16, 20000), _log(rng, 2, 80) * 64, _log(rng, 2, 80) * 256])
        return {"op": op, "x": rng.choice(sorted(X)), "h": rng.choice(sorted(X)), "o": rng.choice(sorted(X)),
                "rows": _log(rng, 1, max(2, min(8192, 8192 * 2000 // cols))), "cols": cols,
                "kind": rng.choice(["rms", "rms", "layer"]), "post": rng.random() < 0.4,
                "gate": rng.choice(["none", "channel", "row", "full"]), "sigmoid": rng.random() < 0.5,
                "scale": rng.choice([1.0, 0.5, 0.22])}
    vocab, n_seq, hi = _log(rng, 1000, 152064), _log(rng, 1, 256), rng.choice([0, 0, 4, 8])
    n_seq = max(1, min(n_seq, 30_000_000 // (vocab * (1 + hi))))
    hist = _log(rng, 1, 32000)
    return {"op": op, "x": rng.choice(["F32", "F32", "F16", "BF16"]), "n_seq": n_seq, "drafts_min": rng.randint(0, hi),
            "drafts_max": hi, "mix": mix, "vocab": vocab, "hist_min": rng.choice([0, hist // 10, hist]),
            "hist_max": hist, "bias": rng.choice([0, 4, 100, 300]), "mask": rng.random() < 0.5}


def lengths(case):
    """Two numbers of each sequence: new tokens and tokens held before (logits: rows and length of the history)."""
    r = random.Random(case["mix"])

    def one(lo, hi):
        if hi <= lo:
            return lo
        return max(lo, min(hi, int(round(math.exp(r.uniform(math.log(lo + 1), math.log(hi + 1))) - 1))))

    if case["op"] == "logits":
        return [(1 + r.randint(case["drafts_min"], case["drafts_max"]), one(case["hist_min"], case["hist_max"]))
                for _ in range(case["n_seq"])]
    got = [(one(case["new_min"], case["new_max"]), one(case["ctx_min"], case["ctx_max"])) for _ in range(case["n_seq"])]
    if case["op"] == "plan":
        for s in r.sample(range(case["n_seq"]), case["ended"]):
            got[s] = (-1, got[s][1])
    return got


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _sums(v):
    out = [0]
    for n in v:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    st = {"case": case}
    {"plan": prepare_plan, "rope": prepare_rope, "norm": prepare_norm, "logits": prepare_logits}[case["op"]](st, g)
    if own:
        import_library(st)
    return st


def prepare_plan(st, g):
    case = st["case"]
    sizes, P = lengths(case), case["page"]
    # a sequence holds the pages of its tokens, now and then one more (its last drafts were not taken)
    held = [-(-ctx // P) + (1 if s % 5 == 3 else 0) for s, (_, ctx) in enumerate(sizes)]
    after = [max(h, -(-(ctx + max(n, 0)) // P)) for h, (n, ctx) in zip(held, sizes)]
    R, W = sum(after) + 7, max(after) + 2
    order = torch.randperm(R, generator=g, device=DEV).to(torch.int32)
    used = sum(held)
    table = torch.full((len(sizes), W), -1, dtype=torch.int32, device=DEV)
    rank = torch.arange(W, device=DEV)
    first = _ints(_sums(held)[:-1])
    pages = _ints(held)
    table = torch.where(rank < pages[:, None], order[(first[:, None] + rank).clamp(max=R - 1).long()], table)
    # the free pages lie in a ring from some place on
    at = int(torch.randint(0, R, (1,), generator=g, device=DEV))
    ring = torch.full((R,), -1, dtype=torch.int32, device=DEV)
    ring[(at + torch.arange(R - used, device=DEV)) % R] = order[used:]
    st.update(held=_ints([c for _, c in sizes]), new=_ints([n for n, _ in sizes]), pages=pages, table=table.contiguous(),
              ring=ring, free=_ints([at, R - used, 0]), T=sum(max(n, 0) for n, _ in sizes) + 3)


def scaling(case):
    """How the frequencies are stretched for contexts longer than those of the training."""
    return {"none": {}, "linear": {"factor": 4.0}, "ntk": {"factor": 8.0}, "yarn": {"factor": 4.0, "original": 32768},
            "bands": {"factor": 8.0, "original": 8192, "low": 1.0, "high": 4.0}}[case["scaling"]]


THETA = 1000000.0


def frequencies(case):
    """Radians a position of each pair, in 64 bits, and the factor of the rotated values."""
    n, kind, s = case["n_rot"], case["scaling"], scaling(case)
    i = torch.arange(n // 2, dtype=torch.float64, device=DEV)
    theta = THETA * s["factor"] ** (n / (n - 2)) if kind == "ntk" else THETA
    f = theta ** (-2.0 * i / n)
    if kind == "linear":
        return f / s["factor"], 1.0
    if kind == "yarn":
        lo, hi = (n * math.log(s["original"] / (turns * 2 * math.pi)) / (2 * math.log(THETA)) for turns in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n - 1)
        slow = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - slow) + f / s["factor"] * slow, 0.1 * math.log(s["factor"]) + 1
    if kind == "bands":
        fast = ((s["original"] * f / (2 * math.pi) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        return f * fast + f / s["factor"] * (1 - fast), 1.0
    return f, 1.0


def prepare_rope(st, g):
    case = st["case"]
    sizes, P, kv, D = lengths(case), case["page"], case["kv_heads"], case["dim"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    starts = _sums(n for n, _ in sizes)
    T = starts[-1]
    held = [-(-(n + ctx) // P) for n, ctx in sizes]
    n_pages, W = sum(held) + 3, max(held) + 1
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    rank = torch.arange(W, device=DEV)
    where = (_ints(_sums(held)[:-1])[:, None] + rank).clamp(max=n_pages - 1)
    table = torch.where(rank < _ints(held)[:, None], order[where], 0).to(torch.int32).contiguous()
    st.update(T=T, start=_ints(starts), len=_ints([n + ctx for n, ctx in sizes]), table=table)
    shape = (n_pages, kv, P, D)
    for name in ("k", "v"):
        x = randn(*shape)
        scaled = case["c"] == "E4M3"
        st[name + "_cache"] = ((120 * x).clamp(-448, 448) if scaled else x).to(C[case["c"]])
        st[name + "_scale"] = torch.exp(0.3 * randn(*shape[:3])) / 120 if scaled else None
    # rows of one fused product: queries, keys and values of a token are next to each other
    st["qkv"] = torch.empty(T, case["heads"] + 2 * kv, D, dtype=X[case["x"]], device=DEV)
    # keys have channels that are larger than the rest, as trained models' do
    st["qkv"].copy_(randn(T, case["heads"] + 2 * kv, D) * torch.exp(0.5 * randn(1, case["heads"] + 2 * kv, D)))
    st["q_weight"], st["k_weight"] = ((1 + 0.3 * randn(D), 1 + 0.3 * randn(D)) if case["norm"] else (None, None))
    st["frequency"], st["factor"] = frequencies(case)


def prepare_norm(st, g):
    case = st["case"]
    T, D = case["rows"], case["cols"]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    # a residual stream has a few channels far above the others
    channel = torch.exp(randn(D)) * torch.where(torch.rand(D, generator=g, device=DEV) < 0.002, 30.0, 1.0)
    st["h"] = (randn(T, D) * channel + (0.3 if case["kind"] == "layer" else 0.0)).to(X[case["h"]])
    st["y"] = (randn(T, D) * torch.exp(0.5 * randn(D))).to(X[case["x"]])
    shape = {"none": None, "channel": (D,), "row": (T,), "full": (T, D)}[case["gate"]]
    st["gate"] = None if shape is None else randn(*shape).to(X[case["x"]] if case["gate"] == "full" else torch.float32)
    layer = case["kind"] == "layer"
    for name in ("pre", "post"):
        there = name == "pre" or case["post"]
        st[name + "_weight"] = 1 + 0.2 * randn(D) if there else None
        st[name + "_bias"] = 0.1 * randn(D) if there and layer else None
    st["h_out"] = torch.empty_like(st["h"])


def prepare_logits(st, g):
    case = st["case"]
    sizes, V = lengths(case), case["vocab"]
    starts, hist = _sums(n for n, _ in sizes), _sums(h for _, h in sizes)
    S, T, H = len(sizes), starts[-1], hist[-1]

    def rand(*shape):
        return torch.rand(shape, generator=g, device=DEV)

    def tokens(n):  # a few tokens come often, as in texts
        return (V * rand(n) ** 6).to(torch.int32).clamp(max=V - 1)

    st.update(T=T, start=_ints(starts), history_start=_ints(hist), history=tokens(H), tokens=tokens(T))
    st["logits"] = (3.0 * torch.randn((T, V), generator=g, device=DEV)).to(X[case["x"]])
    st["prompt"] = (rand(S) * _ints([h for _, h in sizes])).to(torch.int32)
    st.update(repetition=1.0 + 0.3 * rand(S), frequency=0.3 * rand(S), presence=0.5 * rand(S))
    n = case["bias"]
    if n:
        b = [random.Random(case["mix"] + s).randint(0, n) for s in range(S)]
        st["bias_start"] = _ints(_sums(b))
        st["bias_token"] = torch.randint(0, V, (sum(b),), generator=g, device=DEV, dtype=torch.int32)
        st["bias_value"] = 5.0 * torch.randn((sum(b),), generator=g, device=DEV)
    if case["mask"]:
        # one row in four is free; a grammar allows a few hundred tokens, or nearly all
        n_masks, words = max(1, T // 2), (V + 31) // 32
        few = torch.randint(-2 ** 31, 2 ** 31, (n_masks, words), generator=g, device=DEV)
        thin = torch.randint(-2 ** 31, 2 ** 31, (n_masks, words), generator=g, device=DEV)
        st["mask"] = torch.where(torch.arange(n_masks, device=DEV)[:, None] % 2 == 0, few & thin, few | thin).to(torch.int32)
        st["mask_of"] = torch.where(rand(T) < 0.25, -1, torch.randint(0, n_masks, (T,), generator=g, device=DEV)).to(torch.int32)


def import_library(st):
    """The library's handle, and the objects that its user keeps from step to step."""
    sys.path.insert(0, os.path.join(os.getcwd(), "tinycoder-inference_amd"))
    import tc_hip
    case, st["lib"] = st["case"], tc_hip.Library()
    if case["op"] == "plan":
        st["plan"] = tc_hip.KVPlan(st["new"], st["held"], st["pages"], st["table"], st["ring"], st["free"], case["page"], st["T"])
    elif case["op"] == "rope":
        st["cache"] = tc_hip.KVCache(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"])
        st["batch"] = tc_hip.KVBatch(st["start"], st["len"], st["table"])
        st["rope"] = tc_hip.Rope(case["n_rot"], THETA, layout=case["layout"], scaling=case["scaling"], **scaling(case))
    elif case["op"] == "norm":
        st["pre"], st["post"] = (tc_hip.Norm(st[n + "_weight"], st[n + "_bias"], eps=EPS, kind=case["kind"])
                                 if st[n + "_weight"] is not None else None for n in ("pre", "post"))
        st["gate_given"] = st["gate"][:, None] if case["gate"] == "row" else st["gate"]
    elif case["op"] == "logits":
        names = ("repetition", "frequency", "presence", "history", "history_start", "prompt", "bias_start", "bias_token",
                 "bias_value", "mask", "mask_of")
        st["rules"] = tc_hip.LogitRules(**{n: st.get(n) for n in names})


EPS = 1e-6


def run(st):
    return (run_own if own else run_plain)(st)


def run_own(st):
    case, lib = st["case"], st["lib"]
    if case["op"] == "plan":
        p = lib.kv_plan(st["plan"])
        return [p.start, p.length, p.pages_out, p.free_out, p.sequence, p.position, p.slot, p.table, p.ring]
    if case["op"] == "rope":
        H, kv = case["heads"], case["kv_heads"]
        q, k, v = st["qkv"][:, :H], st["qkv"][:, H:H + kv], st["qkv"][:, H + kv:]
        out = lib.rope_kv_write(st["cache"], st["batch"], st["rope"], q, k, v, q_norm=st["q_weight"],
                                k_norm=st["k_weight"], eps=EPS)
        return [out] + cache_of(st)
    if case["op"] == "norm":
        h, x = lib.norm_add(st["h"], st["y"], pre=st["pre"], post=st["post"], gate=st["gate_given"], sigmoid=case["sigmoid"],
                            scale=case["scale"], out_dtype=X[case["o"]], h_out=st["h_out"])
        return [h, x]
    return lib.logits_adjust(st["rules"], st["logits"], st["start"], tokens=st["tokens"])


def cache_of(st):
    return [st[n] for n in ("k_cache", "v_cache", "k_scale", "v_scale") if st[n] is not None]


# ---- the plain forms -----------------------------------------------------------------------------------------------


def run_plain(st):
    return {"plan": plain_plan, "rope": plain_rope, "norm": plain_norm, "logits": plain_logits}[st["case"]["op"]](st)


def plain_plan(st):
    P, T, ring, table = st["case"]["page"], st["T"], st["ring"], st["table"]
    S, W, R = *table.shape, ring.numel()
    held, new, pages = st["held"].long(), st["new"].long(), st["pages"].long()
    ended = new < 0
    start = torch.zeros(S + 1, dtype=torch.long, device=DEV)
    start[1:] = torch.cumsum(new.clamp(min=0), 0)
    start = start.clamp(max=T)
    length = torch.where(ended, 0, held + start[1:] - start[:-1])
    rank = torch.arange(W, device=DEV)
    # pages of ended sequences go behind the free ones; a place past the ring takes what is not to be written
    back = torch.where(ended, pages, 0)
    at, left = st["free"][0].long(), st["free"][1].long()
    place = (at + left + (torch.cumsum(back, 0) - back)[:, None] + rank) % R
    longer = torch.cat([ring, ring[:1]])
    longer.scatter_(0, torch.where(rank < back[:, None], place, R).reshape(-1), table.reshape(-1))
    ring.copy_(longer[:R])
    left = left + back.sum()
    need = (length + P - 1) // P
    want = torch.where(ended, 0, (need.clamp(max=W) - pages).clamp(min=0))
    before = torch.cumsum(want, 0) - want
    j = before[:, None] + rank - pages[:, None]
    given = (rank >= pages[:, None]) & (rank < (pages + want)[:, None])
    table.copy_(torch.where(given, torch.where(j < left, ring[(at + j) % R], -1), table))
    got = torch.minimum(want, left - before).clamp(min=0)
    taken = got.sum()
    missing = want.sum() - taken + (need - need.clamp(max=W)).sum()
    pages = torch.where(ended, 0, pages + got)
    rows = torch.arange(T, device=DEV)
    seq = (torch.searchsorted(start, rows, right=True) - 1).clamp(max=S - 1)
    there = rows < start[-1]
    pos = held[seq] + rows - start[seq]
    page = table[seq, (pos // P).clamp(max=W - 1)].long()
    slot = torch.where(there & (pos // P < W) & (page >= 0), page * P + pos % P, -1)
    return [start.int(), length.int(), pages.int(), torch.stack([(at + taken) % R, left - taken, missing]).int(),
            torch.where(there, seq, -1).int(), torch.where(there, pos, -1).int(), slot, table, ring]


def plain_rope(st):
    case = st["case"]
    H, kv, P, n = case["heads"], case["kv_heads"], case["page"], case["n_rot"]
    rows = torch.arange(st["T"], device=DEV, dtype=torch.int32)
    seq = torch.searchsorted(st["start"], rows, right=True) - 1
    pos = (st["len"][seq] - st["start"][seq + 1] + rows).long()
    a = pos.double()[:, None] * st["frequency"]
    cos, sin = (torch.cos(a) * st["factor"]).float()[:, None], (torch.sin(a) * st["factor"]).float()[:, None]

    def normed(x, weight):
        return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight

    def rotated(x):
        out = x.clone()
        one, two = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
        u, v = x[..., one], x[..., two]
        out[..., one], out[..., two] = u * cos - v * sin, u * sin + v * cos
        return out

    x = st["qkv"].float()
    q, k = rotated(normed(x[:, :H], st["q_weight"])), rotated(normed(x[:, H:H + kv], st["k_weight"]))
    page, slot = st["table"][seq, pos // P].long(), pos % P
    plain_store(st, "k", k, page, slot)
    plain_store(st, "v", x[:, H + kv:], page, slot)
    return [q.to(X[case["x"]])] + cache_of(st)


def plain_store(st, name, x, page, slot):
    cache = st[name + "_cache"]
    if st[name + "_scale"] is None:
        cache[page, :, slot] = x.to(cache.dtype)
        return
    d = x.abs().amax(-1)
    d = d / torch.full_like(d, 448.0)
    d = torch.where(d == 0, torch.ones_like(d), d)
    st[name + "_scale"][page, :, slot] = d
    # (assignment by index is not there for this type)
    cache.view(torch.uint8)[page, :, slot] = (x / d[..., None]).clamp(-448, 448).to(cache.dtype).view(torch.uint8)


def plain_norm(st):
    case = st["case"]

    def normed(x, name):
        if case["kind"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * st[name + "_weight"]
        return x if st[name + "_bias"] is None else x + st[name + "_bias"]

    y = st["y"].float()
    if case["post"]:
        y = normed(y, "post")
    if st["gate"] is not None:
        gate = st["gate"].float()
        gate = torch.sigmoid(gate) if case["sigmoid"] else gate
        y = y * (gate[:, None] if case["gate"] == "row" else gate)
    h = st["h"].float() + case["scale"] * y
    st["h_out"].copy_(h)
    return [st["h_out"], normed(h, "pre").to(X[case["o"]])]


def plain_logits(st):
    case, T = st["case"], st["T"]
    V, S = case["vocab"], case["n_seq"]
    rows = torch.arange(T, device=DEV)
    start = st["start"].long()
    seq = torch.searchsorted(start, rows, right=True) - 1
    h = torch.arange(st["history"].numel(), device=DEV)
    of = torch.searchsorted(st["history_start"].long(), h, right=True) - 1
    answer = h - st["history_start"][of] >= st["prompt"][of]
    at = of * V + st["history"]
    seen = torch.zeros(S * V, device=DEV).index_fill_(0, at, 1.0).reshape(S, V)[seq]
    count = torch.zeros(S * V, device=DEV).index_add_(0, at, answer.float()).reshape(S, V)[seq]
    # row i of a sequence also counts its chunk's tokens up to the i-th
    back = torch.arange(case["drafts_max"] + 1, device=DEV)
    earlier = rows[:, None] - back
    token = st["tokens"][earlier.clamp(min=0)].long()
    count.scatter_add_(1, token, (earlier >= start[seq][:, None]).float())
    x = st["logits"].float()
    rep = st["repetition"][seq][:, None]
    x = torch.where((seen + count) > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - st["frequency"][seq][:, None] * count - st["presence"][seq][:, None] * (count > 0)
    if case["bias"]:
        b = torch.arange(st["bias_token"].numel(), device=DEV)
        of = torch.searchsorted(st["bias_start"].long(), b, right=True) - 1
        bias = torch.zeros(S * V, device=DEV).index_add_(0, of * V + st["bias_token"], st["bias_value"]).reshape(S, V)
        x = x + bias[seq]
    if case["mask"]:
        v = torch.arange(V, device=DEV)
        words = st["mask"][st["mask_of"].clamp(min=0).long()]
        bit = (words[:, v // 32] >> (v % 32)) & 1
        x = torch.where((bit == 0) & (st["mask_of"] >= 0)[:, None], -math.inf, x)
    return x


# ---- the same from the definitions in 64 bits ----------------------------------------------------------------------


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    st = prepare(case, seed)
    return {"rope": exact_rope, "norm": exact_norm, "logits": exact_logits}[case["op"]](st)


def exact_rope(st):
    case, sizes = st["case"], lengths(st["case"])
    H, kv, P, D, n = case["heads"], case["kv_heads"], case["page"], case["dim"], case["n_rot"]
    where = [ctx + i for new, ctx in sizes for i in range(new)]
    of = [s for s, (new, _) in enumerate(sizes) for _ in range(new)]
    table = st["table"].tolist()
    page = torch.tensor([table[s][p // P] for s, p in zip(of, where)], device=DEV)
    slot = torch.tensor([p % P for p in where], device=DEV)
    turn = torch.polar(torch.full((len(where), n // 2), st["factor"], dtype=torch.float64, device=DEV),
                       torch.tensor(where, dtype=torch.float64, device=DEV).outer(st["frequency"]))
    x = st["qkv"].double()

    def head(h, weight):
        r = x[:, h]
        if weight is not None:
            r = r / (r.square().sum(1, keepdim=True) / D + EPS).sqrt() * weight.double()
        if case["layout"] == "half":
            z = torch.complex(r[:, :n // 2].contiguous(), r[:, n // 2:n].contiguous()) * turn
            return torch.cat([z.real, z.imag, r[:, n:]], 1)
        z = torch.complex(r[:, 0:n:2].contiguous(), r[:, 1:n:2].contiguous()) * turn
        return torch.cat([torch.view_as_real(z).reshape(len(where), n), r[:, n:]], 1)

    out = [torch.stack([head(h, st["q_weight"]) for h in range(H)], 1)]
    rows = {"k": torch.stack([head(H + h, st["k_weight"]) for h in range(kv)], 1), "v": x[:, H + kv:]}
    scales = []
    for name in ("k", "v"):
        cache, r = st[name + "_cache"].double(), rows[name]
        if st[name + "_scale"] is not None:
            d = r.abs().amax(-1) / 448
            scale = st[name + "_scale"].double()
            scale[page, :, slot] = d
            scales.append(scale)
            r = r / d[..., None]
        cache[page, :, slot] = r
        out.append(cache)
    return out + scales


def exact_norm(st):
    case = st["case"]
    D = case["cols"]

    def normed(x, name):
        m = x.sum(1) / D if case["kind"] == "layer" else torch.zeros_like(x[:, 0])
        var = (x - m[:, None]).square().sum(1) / D
        z = (x - m[:, None]) / (var + EPS).sqrt()[:, None] * st[name + "_weight"].double()
        return z if st[name + "_bias"] is None else z + st[name + "_bias"].double()

    y = st["y"].double()
    if case["post"]:
        y = normed(y, "post")
    if st["gate"] is not None:
        gate = st["gate"].double()
        if case["sigmoid"]:
            gate = 1 / (1 + torch.exp(-gate))
        y = y * gate.reshape(-1, 1) if case["gate"] == "row" else y * gate
    h = st["h"].double() + case["scale"] * y
    return [h, normed(h, "pre")]


def exact_logits(st):
    case, sizes = st["case"], lengths(st["case"])
    V = case["vocab"]
    out = torch.empty(st["T"], V, dtype=torch.float64, device=DEV)
    history, tokens = st["history"].cpu(), st["tokens"].cpu()
    t = h = 0
    bias_at = st["bias_start"].tolist() if case["bias"] else None
    bits = torch.arange(32, device=DEV)
    for s, (n, length) in enumerate(sizes):
        prompt = int(st["prompt"][s])
        seen = torch.bincount(history[h:h + length].long(), minlength=V)
        count = torch.bincount(history[h + prompt:h + length].long(), minlength=V)
        rep, freq, pres = (float(st[name][s]) for name in ("repetition", "frequency", "presence"))
        bias = torch.zeros(V, dtype=torch.float64, device=DEV)
        if case["bias"]:
            part = slice(bias_at[s], bias_at[s + 1])
            bias.index_add_(0, st["bias_token"][part].long(), st["bias_value"][part].double())
        for i in range(n):
            seen[tokens[t + i]] += 1
            count[tokens[t + i]] += 1
            x = st["logits"][t + i].double()
            c = count.to(DEV).double()
            x = torch.where(seen.to(DEV) > 0, torch.where(x > 0, x / rep, x * rep), x) - freq * c - pres * (c > 0) + bias
            if case["mask"] and int(st["mask_of"][t + i]) >= 0:
                word = st["mask"][int(st["mask_of"][t + i])].long()
                allowed = ((word[:, None] >> bits) & 1).reshape(-1)[:V] == 1
                x = x.masked_fill(~allowed, -math.inf)
            out[t + i] = x
        t, h = t + n, h + length
    return out


def work(case):
    op = case["op"]
    if op == "norm":
        T, D, e = case["rows"], case["cols"], {"F32": 4, "F16": 2, "BF16": 2}
        weights = (1 + case["post"]) * (2 if case["kind"] == "layer" else 1) * 4 * D
        gate = {"none": 0, "channel": 4 * D, "row": 4 * T, "full": e[case["x"]] * T * D}[case["gate"]]
        return {"bytes": T * D * (e[case["x"]] + 2 * e[case["h"]] + e[case["o"]]) + weights + gate,
                "flops": T * D * (8 + 4 * case["post"])}
    sizes = lengths(case)
    T, S = sum(max(n, 0) for n, _ in sizes), len(sizes)
    if op == "plan":
        P = case["page"]
        pages = sum(-(-ctx // P) if n < 0 else -(-(ctx + n) // P) - -(-ctx // P) for n, ctx in sizes)
        return {"bytes": 24 * S + 8 * pages + 16 * T, "flops": 4 * (S + T)}
    if op == "rope":
        x, D, kv = (4 if case["x"] == "F32" else 2), case["dim"], case["kv_heads"]
        row = D + 4 if case["c"] == "E4M3" else 2 * D  # one cached key or value of a head
        return {"bytes": T * (2 * case["heads"] * D * x + 2 * kv * (D * x + row)),
                "flops": 3 * T * (case["heads"] + kv) * case["n_rot"]}
    V = case["vocab"]
    masks = T * 3 // 4 * (V // 8) if case["mask"] else 0
    return {"bytes": T * V * (4 + (4 if case["x"] == "F32" else 2)) + masks + 4 * sum(h for _, h in sizes),
            "flops": 3 * T * V}
