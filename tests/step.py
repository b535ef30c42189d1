"""The operators around a step's products and attention (tc_step.h) from their definitions, in
Python's integers and 64 bits, for the tests of tc_kv_plan, tc_rope_*, tc_norm_add and tc_logits_adjust."""
import math

import numpy as np
import torch

DT = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
# half a step of a rounding, relative to the value, and the least half step (of subnormal numbers)
HALF = {"F32": 2.0 ** -24, "F16": 2.0 ** -11, "BF16": 2.0 ** -8}
LEAST = {"F32": 2.0 ** -150, "F16": 2.0 ** -25, "BF16": 2.0 ** -134}
U = 2.0 ** -24  # an fp32 rounding


def tensor(a, dev, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev) if dtype is None else torch.from_numpy(np.ascontiguousarray(a)).to(dtype).to(dev)


def f64(t):
    return t.detach().double().cpu().numpy()


# ---- plan ------------------------------------------------------------------------------------------------------------


def plan_exact(new, held, pages, table, ring, free, page, n_tokens):
    """One step by hand: a dict of everything tc_kv_plan writes (table and ring as copies)."""
    S, W, R = len(new), table.shape[1], len(ring)
    table, ring = table.copy(), ring.copy()
    at, left = min(max(int(free[0]), 0), R - 1), min(max(int(free[1]), 0), R)
    for s in range(S):
        if new[s] < 0:
            for j in range(min(max(int(pages[s]), 0), W)):
                if left < R:
                    ring[(at + left) % R] = table[s, j]
                    left += 1
    start, length, pages_out = [0], [], []
    missing = 0
    for s in range(S):
        rows = min(max(int(new[s]), 0), n_tokens - start[-1])
        start.append(start[-1] + rows)
        if new[s] < 0:
            length.append(0)
            pages_out.append(0)
            continue
        length.append(min(max(int(held[s]), 0) + rows, 2 ** 31 - 65))
        n = min(max(int(pages[s]), 0), W)
        need = -(-length[-1] // page)
        got = n
        for j in range(n, min(need, W)):
            if left:
                table[s, j] = ring[at]
                at, left, got = (at + 1) % R, left - 1, got + 1
            else:
                table[s, j] = -1
                missing += 1
        missing += max(0, need - W)
        pages_out.append(got)
    seq, pos, slot = [-1] * n_tokens, [-1] * n_tokens, [-1] * n_tokens
    for s in range(S):
        for t in range(start[s], start[s + 1]):
            p = length[s] - (start[s + 1] - start[s]) + t - start[s]
            seq[t], pos[t] = s, p
            if p // page < W and table[s, p // page] >= 0:
                slot[t] = int(table[s, p // page]) * page + p % page
    i32 = np.int32
    return dict(start=np.array(start, i32), length=np.array(length, i32), pages_out=np.array(pages_out, i32),
                free_out=np.array([at, left, min(missing, 2 ** 30)], i32), sequence=np.array(seq, i32),
                position=np.array(pos, i32), slot=np.array(slot, np.int64), table=table, ring=ring)


# ---- rotary positions ------------------------------------------------------------------------------------------------


def turns_exact(n_rot, theta, scaling="none", factor=1.0, original=0.0, low=0.0, high=0.0, divisors=None):
    """(turns a position of each pair, the factor of the values)."""
    out, m = [], 1.0
    if scaling == "ntk":
        theta = theta * factor ** (n_rot / (n_rot - 2))
    for i in range(n_rot // 2):
        f = theta ** (-2.0 * i / n_rot)
        if scaling == "linear":
            f /= factor
        elif scaling == "yarn":
            lo, hi = low or 1.0, high or 32.0
            a = max(math.floor(n_rot * math.log(original / (hi * 2 * math.pi)) / (2 * math.log(theta))), 0)
            b = min(math.ceil(n_rot * math.log(original / (lo * 2 * math.pi)) / (2 * math.log(theta))), n_rot - 1)
            r = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f = f * (1 - r) + f / factor * r
            m = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
        elif scaling == "bands":
            r = min(max((original * f / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f = f * r + f / factor * (1 - r)
        out.append(f / (2 * math.pi) / (float(divisors[i]) if divisors is not None else 1.0))
    return np.array(out), m


def rope_exact(x, pos, turns, n_rot, layout, factor, norm=None, eps=1e-6):
    """x fp64 [T][heads][D] at positions: (out, how far fp32 work may be from it, before the last rounding).

    cos and sin are off by 2^-23, the factor's product, the pair's product and its sum by a rounding each. A norm
    multiplies by 1/sqrt: a sum of D positive squares (each lane 8 of them one after the other, then 5 steps of a
    tree: 15 roundings with the mean and eps, half of them behind the root), the root's 2 and two products: 12 at most."""
    T, H, D = x.shape
    off = np.zeros_like(x)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm
        off = np.abs(x) * 12 * U
    a = 2 * np.pi * np.modf(pos[:, None].astype(np.float64) * turns)[0]
    c, s = (np.cos(a) * factor)[:, None], (np.sin(a) * factor)[:, None]
    one = np.arange(n_rot // 2) if layout == "half" else 2 * np.arange(n_rot // 2)
    two = one + (n_rot // 2 if layout == "half" else 1)
    out, mass = x.copy(), np.abs(x)
    u, v = x[..., one], x[..., two]
    out[..., one], out[..., two] = u * c - v * s, u * s + v * c
    big = (np.abs(u) + np.abs(v)) * abs(factor)
    err = off.copy()
    err[..., one] = err[..., two] = big * 5 * U + (off[..., one] + off[..., two]) * abs(factor)
    return out, err


# ---- norms -----------------------------------------------------------------------------------------------------------


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-x))


def norm_exact(z, err, weight, bias, eps, kind, offset):
    """(norm of rows z, how far fp32 work on rows that are off by err may be from it).

    A sum over a row: 32 values of a lane at most, one after the other, 6 steps over a wave, 6 over the waves, the
    mean's product: 45 roundings, each of at most the sum of magnitudes."""
    n = 45
    if kind == "layer":
        mean = z.mean(1, keepdims=True)
        err = err + np.abs(z - mean) * U + (np.abs(z).mean(1, keepdims=True) * n * U + err.mean(1, keepdims=True))
        z = z - mean
    sq = (z * z).mean(1, keepdims=True) + eps
    # of the mean square: its roundings, and what the rows' own errors make (relative, twice the weighted mean)
    rel = (n + 2) * U + 2 * np.sqrt((err * err).mean(1, keepdims=True) / sq)
    inv = 1 / np.sqrt(sq)
    w = 1.0 if weight is None else weight + offset
    out = z * inv * w
    off = np.abs(w) * inv * (err + np.abs(z) * (rel / 2 + 4 * U)) + np.abs(z) * inv * U * (np.abs(w) if weight is not None else 0)
    if bias is not None:
        out = out + bias
        off = off + np.abs(out) * U
    return out, off * 1.01


def norm_add_exact(h, y, pre, post, gate, sig, scale):
    """pre, post: None or (weight, bias, eps, kind, offset); gate: None or broadcast to h. -> (h', its error, x, its
    error), before the last roundings."""
    if y is not None:
        err = np.zeros_like(y)
        if post is not None:
            y, err = norm_exact(y, err, *post)
        g, ge = np.full_like(y, scale), 0.0
        if gate is not None:
            s = sigmoid(gate) if sig else gate
            # exp of an fp32 number 2 steps off at most, its sum and quotient: 6 roundings
            g, ge = s * scale, (6 * U if sig else 0.0) + U
        err = np.abs(g) * err + np.abs(g * y) * (ge + U)
        h = h + g * y
        err = err + np.abs(h) * U
    else:
        err = np.zeros_like(h)
    if pre is None:
        return h, err, None, None
    return (h, err) + norm_exact(h, err, *pre)


# ---- rules on logits -------------------------------------------------------------------------------------------------


def logits_exact(l, start, tokens=None, repetition=None, frequency=None, presence=None, history=None, history_start=None,
                 prompt=None, bias_start=None, bias_token=None, bias_value=None, mask=None, mask_of=None):
    """l fp64 [T][V]; rows past the last sequence are NaN in the result."""
    T, V = l.shape
    out = np.full((T, V), np.nan)
    S = len(start) - 1
    for s in range(S):
        rep, freq, pres = (float(a[s]) if a is not None else d for a, d in ((repetition, 1.0), (frequency, 0.0), (presence, 0.0)))
        seen, answered = set(), {}
        if history is not None:
            part = history[history_start[s]:history_start[s + 1]]
            for i, t in enumerate(part):
                if 0 <= t < V:
                    seen.add(int(t))
                    if prompt is None or i >= prompt[s]:
                        answered[int(t)] = answered.get(int(t), 0) + 1
        bias = {}
        if bias_start is not None:
            for i in range(bias_start[s], bias_start[s + 1]):
                t = int(bias_token[i])
                bias[t] = np.float32(np.float32(bias.get(t, 0.0)) + np.float32(bias_value[i]))
        for r in range(start[s], start[s + 1]):
            if tokens is not None and 0 <= tokens[r] < V:
                seen.add(int(tokens[r]))
                answered[int(tokens[r])] = answered.get(int(tokens[r]), 0) + 1
            x = l[r].copy()
            for t in seen:
                x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            for t, c in answered.items():
                x[t] -= freq * c + pres
            for t, b in bias.items():
                if 0 <= t < V:
                    x[t] += float(b)
            if mask is not None:
                m = r if mask_of is None else mask_of[r]
                if 0 <= m < len(mask):
                    bits = np.unpackbits(mask[m].view(np.uint8), bitorder="little")[:V]
                    x[bits == 0] = -np.inf
            out[r] = x
    return out
