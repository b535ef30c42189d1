"""Paged caches with batches over them, and the operators on them in 64 bits, for
the tests of tc_kv_write, tc_kv_read and tc_attn."""
import numpy as np
import torch

DT = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16, "I8": torch.int8, "E4M3": torch.float8_e4m3fn}
# half a step of a rounding, relative to the value
HALF = {"F32": 2.0 ** -24, "F16": 2.0 ** -11, "BF16": 2.0 ** -8, "E4M3": 2.0 ** -4}
TOP = {"I8": 127.0, "E4M3": 448.0}


def scaled(ctype):
    return ctype in TOP


class Batch:
    """Sequences of (new rows, length in the cache); pages in a random order."""

    def __init__(self, rng, seqs, page, kv_heads, dim, ctype, pad_rows=0, spare=2, width=None):
        self.seqs, self.page, self.kv_heads, self.dim, self.ctype = seqs, page, kv_heads, dim, ctype
        self.start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.length = np.array([total for _, total in seqs], np.int32)
        held = [max(0, -(-total // page)) for _, total in seqs]
        self.n_pages = sum(held) + spare
        width = width or max(held + [1])
        order = rng.permutation(self.n_pages).astype(np.int32)
        # entries behind a sequence's pages are never to be followed
        self.table = np.full((len(seqs), width), -1, np.int32)
        at = 0
        for s, h in enumerate(held):
            self.table[s, :min(h, width)] = order[at:at + min(h, width)]
            at += h
        self.T = int(self.start[-1]) + pad_rows
        shape = (self.n_pages, kv_heads, page, dim)
        self.host = {}
        for name in ("k", "v"):
            if ctype == "I8":
                c = torch.from_numpy(rng.integers(-127, 128, shape).astype(np.int8))
            elif ctype == "E4M3":
                c = torch.from_numpy((150 * rng.standard_normal(shape)).clip(-448, 448).astype(np.float32)).to(DT[ctype])
            else:
                c = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(DT[ctype])
            self.host[name] = c
            if scaled(ctype):
                self.host[name + "_scale"] = torch.from_numpy(
                    (np.exp(0.5 * rng.standard_normal(shape[:3])) / (70 if ctype == "I8" else 150)).astype(np.float32))

    def to(self, dev):
        import tc_hip
        self.dev = {n: t.to(dev) for n, t in self.host.items()}
        self.cache = tc_hip.KVCache(self.dev["k"], self.dev["v"], self.dev.get("k_scale"), self.dev.get("v_scale"))
        self.batch = tc_hip.KVBatch(*(torch.from_numpy(a).to(dev) for a in (self.start, self.length, self.table)))
        return self

    def slot(self, s, pos):
        """(page, slot) of a position; None where no page holds it."""
        if pos < 0 or pos // self.page >= self.table.shape[1]:
            return None
        p = int(self.table[s, pos // self.page])
        return (p, pos % self.page) if 0 <= p < self.n_pages else None

    def rows(self):
        """(row, sequence, position) of every row of the batch."""
        for s, (n, total) in enumerate(self.seqs):
            for i in range(n):
                yield int(self.start[s]) + i, s, total - n + i

    def value(self, name, host=None):
        """The whole cache as fp64 values."""
        h = host or self.host
        x = h[name].float().double().numpy()
        return x * h[name + "_scale"].double().numpy()[..., None] if scaled(self.ctype) else x


def attn_exact(b, q, scale, window=0):
    """-> (out, mass, terms, absv): attention of q (fp64 [T][heads][dim]) and, for each output, sum_j p_j |v_j|,
    the largest score error that one rounding of relative size 1 to every term of it would make, and
    sum_j |v_j|."""
    T, H, D = q.shape
    G = H // b.kv_heads
    k, v = b.value("k"), b.value("v")
    out, mass = np.zeros((T, H, D)), np.zeros((T, H, D))
    terms, absv = np.zeros((T, H, 1)), np.zeros((T, H, D))
    for t, s, pos in b.rows():
        lo = max(0, pos - window + 1) if window else 0
        where = [w for w in (b.slot(s, j) for j in range(lo, pos + 1)) if w is not None]
        if not where:
            continue
        pg, sl = (np.array(x) for x in zip(*where))
        for h in range(H):
            K, V = k[pg, h // G, sl], v[pg, h // G, sl]
            z = K @ q[t, h] * scale
            p = np.exp(z - z.max())
            p /= p.sum()
            out[t, h], mass[t, h] = p @ V, p @ np.abs(V)
            absv[t, h] = np.abs(V).sum(0)
            terms[t, h] = (np.abs(K) @ np.abs(q[t, h])).max() * scale
    return out, mass, terms, absv


def attn_bound(xtype, ctype, D, n, out, mass, terms, absv):
    """How far tc_attn may be from the 64-bit result: a score is off by (D + 8) fp32 roundings of its terms
    (products, sums, scale, factor, exponential) and q's own pieces; a weight p by that much twice (its own
    and the sum's score), and by its rounding to the matrix cores' type; the n-term sums by fp32 roundings;
    the output by its own rounding."""
    # what is left of q and p behind their pieces: 1 or 2 of fp16 (11 bits each), 1 to 3 of bf16 (8 bits each)
    piece = {("F32", "BF16"): 2.0 ** -24, ("F16", "BF16"): 2.0 ** -16, ("BF16", "BF16"): 2.0 ** -8,
             ("F32", "F16"): 2.0 ** -22}.get((xtype, "BF16" if ctype == "BF16" else "F16"), 2.0 ** -11)
    # (rows of 16 bits are exact in their pieces)
    q_off = piece if xtype == "F32" else 0.0
    score = terms * ((D + 8) * 2.0 ** -24 + q_off)
    # below fp16's smallest normal number, 2^-14, its step is 2^-24 whatever the value: half of it is not
    # HALF of the value
    least = 2.0 ** -25 if xtype == "F16" else 1e-30
    # weights enter fp16 operands as 2^11 p or more, where the row's largest p is 1: half a step of fp16's
    # subnormals, 2^-25, is 2^-36 of that p, for every token, however small its weight
    if ctype != "BF16":
        least = least + absv * 2.0 ** -36
    return mass * (2.1 * score + piece + (n + 16) * 2.0 ** -24) + HALF[xtype] * np.abs(out) + least
