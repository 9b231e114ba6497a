"""The 8-bit KV cache in numpy: the definition, token by token.

Codes and scales follow float32 as the cache defines them; attention, its
weights and everything else are float64.  Records are read and written by
their byte offsets, one token at a time.
"""
from __future__ import annotations

import math

import numpy as np

from air_amd import capi

UNIT = {capi.KV8_I8: np.float32(1) / np.float32(127), capi.KV8_E4M3: np.float32(1) / np.float32(448)}
BLOCK = 16


def e4m3_values() -> np.ndarray:
    out = np.empty(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        x = math.nan if e == 15 and f == 7 else f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10)
        out[c] = -x if c & 128 else x
    return out


E4M3 = e4m3_values()
_MAGNITUDES = E4M3[:127]          # codes 0..126: 0 .. 448, ascending


def encode(q: np.ndarray, kind: int) -> np.ndarray:
    """Nearest codes (ties to even) of float32 quotients, as stored bytes."""
    q = np.asarray(q, dtype=np.float32).astype(np.float64)
    if kind == capi.KV8_I8:
        return (np.clip(np.rint(q), -127, 127) + 128).astype(np.uint8)
    a = np.clip(np.abs(q), 0.0, 448.0)
    hi = np.searchsorted(_MAGNITUDES, a)                    # first magnitude >= a
    lo = np.maximum(hi - 1, 0)
    up, down = _MAGNITUDES[hi] - a, a - _MAGNITUDES[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)) | (hi == 0), hi, lo)
    return (code + np.where(np.signbit(q), 128, 0)).astype(np.uint8)


def value(code: np.ndarray, kind: int) -> np.ndarray:
    if kind == capi.KV8_I8:
        return code.astype(np.float64) - 128.0
    return E4M3[code]


class Cache:
    """A pool of pages as numpy bytes, with the layout of one call."""

    def __init__(self, kind, kv_heads, head_dim, layers, page_tokens, pool_pages, max_pages, seed=0):
        self.kind, self.kvh, self.d, self.layers = kind, kv_heads, head_dim, layers
        self.page_tokens, self.pool_pages, self.max_pages = page_tokens, pool_pages, max_pages
        self.bpp = page_tokens // BLOCK
        self.record = 128 + 32 * head_dim
        # What earlier users of the pages left: any bytes as codes, finite scales.
        rng = np.random.default_rng(seed)
        self.pool = rng.integers(0, 256, (pool_pages, layers, kv_heads, self.bpp, self.record), dtype=np.uint8)
        self.floats(self.pool)[..., :32] = rng.uniform(0.5, 2.0, self.pool.shape[:-1] + (32,)).astype(np.float32)

    @staticmethod
    def floats(rec):
        return rec.view(np.float32)

    def layout(self, pointer, chunks=None, chunk_shift=0):
        return capi.Kv8Layout(pointer, self.page_tokens, self.kvh, self.d, self.layers, self.max_pages,
                              self.pool_pages, chunks, chunk_shift, self.kind)

    def slot(self, table, layer, head, token):
        """The record of a token and its place in it; None without a page."""
        p = token // self.page_tokens
        if token < 0 or p >= self.max_pages or not 0 <= table[p] < self.pool_pages:
            return None
        return self.pool[table[p], layer, head, token % self.page_tokens // BLOCK], token % BLOCK

    def k_at(self, t):
        dims = np.arange(self.d)
        return 128 + (t // 4 * (self.d // 16) + dims // 16) * 64 + t % 4 * 16 + dims % 16

    def v_at(self, t):
        return 128 + BLOCK * self.d + np.arange(self.d) * BLOCK + t

    def token(self, table, layer, head, token):
        """(k, v, weight) of a token in 64 bits, or None."""
        at = self.slot(table, layer, head, token)
        if at is None:
            return None
        rec, t = at
        f = self.floats(rec)
        return (value(rec[self.k_at(t)], self.kind) * float(f[0]), value(rec[self.v_at(t)], self.kind) * float(f[1]),
                float(f[16 + t]))

    def append(self, qkv, q_width, positions, tables, layer):
        """One call of at most 2048 rows."""
        width = self.kvh * self.d
        blocks = {}
        for r, pos in enumerate(positions):
            if pos >= 0 and self.slot(tables[r], layer, 0, pos) is not None:
                key = (int(tables[r][pos // self.page_tokens]), pos % self.page_tokens // BLOCK)
                blocks.setdefault(key, {})[pos % BLOCK] = r          # the last row of a slot stays
        for (page, block), rows in blocks.items():
            first = min(rows)
            for head in range(self.kvh):
                rec = self.pool[page, layer, head, block]
                f = self.floats(rec)
                for which, at in ((0, self.k_at), (1, self.v_at)):
                    lo = q_width + which * width + head * self.d
                    x = {t: qkv[r, lo:lo + self.d].astype(np.float32) for t, r in rows.items()}
                    top = np.float32(max(np.abs(v).max() if np.isfinite(v).all() else math.inf for v in x.values()))
                    need = top * UNIT[self.kind] if np.isfinite(top) else np.float32(math.nan)
                    old = f[which].copy()
                    scale = need
                    if first > 0:
                        scale = old if np.isnan(old) or need <= old else need
                        if scale != old and not np.isnan(scale):
                            ratio = np.float32(old / scale)
                            for t in range(first):
                                was = value(rec[at(t)], self.kind).astype(np.float32)
                                rec[at(t)] = encode(was * ratio, self.kind)
                    for t, v in x.items():
                        ok = scale > 0
                        rec[at(t)] = encode(v / scale, self.kind) if ok else encode(np.zeros_like(v), self.kind)
                    f[which] = scale
                for t in rows:
                    f[16 + t] = 0.0

    def live(self, table, layer, head, upto):
        """Tokens 0..upto that have a page, with their k, v and scales of v."""
        got = [(t, self.token(table, layer, head, t)) for t in range(upto + 1)]
        got = [(t, x) for t, x in got if x is not None]
        if not got:
            return [], np.zeros((0, self.d)), np.zeros((0, self.d)), np.zeros(0)
        scale = [float(self.floats(self.slot(table, layer, head, t)[0])[1]) for t, _ in got]
        return [t for t, _ in got], np.stack([x[0] for _, x in got]), np.stack([x[1] for _, x in got]), np.array(scale)

    def attention(self, qkv, positions, tables, layer, q_heads, max_tokens, runs=None, weights=None):
        """out, how far a sound f32 computation may be from it, and with
        weights ("add" or "set") the tolerances of the weights it stored."""
        m, group = len(positions), q_heads // self.kvh
        out = np.zeros((m, q_heads, self.d))
        tol = np.zeros((m, q_heads, self.d))
        runs = runs if runs is not None else [(r, r + 1) for r in range(m)]
        far = []
        for begin, end in runs:
            for g in range(self.kvh):
                gathered, slack = {}, {}
                cached = {}
                for r in range(begin, end):
                    upto = min(positions[r], max_tokens - 1)
                    if upto not in cached:
                        cached[upto] = self.live(tables[r], layer, g, upto)
                    tokens, k, v, scale = cached[upto]
                    if not tokens:
                        continue
                    for h in range(g * group, (g + 1) * group):
                        q = qkv[r, h * self.d:(h + 1) * self.d].astype(np.float64)
                        s = k @ q / math.sqrt(self.d)
                        p = np.exp(s - s.max())
                        p /= p.sum()
                        out[r, h] = p @ v
                        ds, rel = self.rounding(q, k, len(tokens))
                        # f16's smallest step is 2^-24 and the call's largest p * scale
                        # lies above 2^13 of its units, so each p * scale is held to
                        # 2^-38 of the largest one at least, times its code (a dim whose
                        # code is zero where p is large sums p's that are tiny).
                        codes = np.abs(v / np.where(scale > 0, scale, 1)[:, None]).sum(axis=0)
                        tol[r, h] = rel * (p @ np.abs(v)) + 2.0 ** -38 * (p * scale).max() * codes + 1e-30
                        for t, x, y in zip(tokens, p, p * rel):
                            gathered[t] = gathered.get(t, 0.0) + x
                            slack[t] = slack.get(t, 0.0) + y
                if weights and end > begin:
                    reach = min(max(positions[begin:end]), max_tokens - 1)
                    for t in range(reach + 1):
                        at = self.slot(tables[begin], layer, g, t)
                        if at is None:
                            continue
                        f = self.floats(at[0])
                        old = float(f[16 + at[1]]) if weights == "add" else 0.0
                        new = old + gathered.get(t, 0.0)
                        rows = group * (end - begin)
                        # The p's own slack, the sum of the rows and the addition.
                        far.append((tables[begin], layer, g, t, slack.get(t, 0.0) + 2.0 ** -24 * (rows + 2) * new))
                        f[16 + at[1]] = new
        return out.reshape(m, -1), tol.reshape(m, -1), far

    def rounding(self, q, k, tokens):
        """Bounds for f32 sums with both operands held to 22 bits, errors of
        the sums growing as a random walk (six standard deviations).

        score: 2 D terms of q k, each rounded to 2^-24 of the running sum, the
               two halves of q hold it to 2^-22 of its largest value, scale
               factors 4 * 2^-24;
        p:     e^s turns the score's error into a relative one, once above
               and once in the denominator; 2^-21 for the exponential, its
               reduced argument and p's two halves;
        sum:   over the tokens, as a random walk."""
        terms = np.abs(k) @ np.abs(q) / math.sqrt(self.d)
        coarse = np.abs(k).sum(axis=1) * np.abs(q).max() / math.sqrt(self.d)
        ds = float((terms * (4 + 6 * math.sqrt(2 * self.d)) * 2.0 ** -24 + coarse * 2.0 ** -23).max())
        return ds, 2 * ds + 2.0 ** -21 + 6 * math.sqrt(tokens) * 2.0 ** -24

    def evict(self, lengths, tables, new_tables, layer, layers, keep_first, keep_last, budget, max_tokens):
        kept = np.full((len(lengths), layers, self.kvh, budget), -1, dtype=np.int32)
        src = self.pool.copy()
        for i, n in enumerate(lengths):
            n = max(0, min(n, max_tokens, self.max_pages * self.page_tokens))
            for l in range(layers):
                for g in range(self.kvh):
                    ids = list(range(n))
                    if n > budget:
                        def rank(t):
                            at = self.slot(tables[i], layer + l, g, t)
                            w = float(self.floats(at[0])[16 + at[1]]) if at is not None else math.nan
                            return (1, 0.0, t) if math.isnan(w) else (0, -w, t)
                        middle = sorted(range(keep_first, n - keep_last), key=rank)
                        ids = sorted(list(range(keep_first)) + middle[:budget - keep_first - keep_last] +
                                     list(range(n - keep_last, n)))
                    kept[i, l, g, :len(ids)] = ids
        if new_tables is tables:
            moved = [i for i, n in enumerate(lengths) if min(n, max_tokens) > budget]
        else:
            moved = range(len(lengths))
        old = Cache.__new__(Cache)
        old.__dict__.update(self.__dict__)
        old.pool = src
        for i in moved:
            for l in range(layers):
                for g in range(self.kvh):
                    ids = [t for t in kept[i, l, g] if t >= 0]
                    for b in range(0, len(ids), BLOCK):
                        at = self.slot(new_tables[i], layer + l, g, b)
                        if at is None:
                            continue
                        rec = at[0]
                        f = self.floats(rec)
                        part = [old.slot(tables[i], layer + l, g, t) for t in ids[b:b + BLOCK]]
                        for which, place in ((0, self.k_at), (1, self.v_at)):
                            scales = [old.floats(p[0])[which] if p is not None else np.float32(0) for p in part]
                            scale = np.float32(math.nan) if any(np.isnan(s) for s in scales) else max(scales)
                            for t, p in enumerate(part):
                                code = encode(np.zeros(self.d, np.float32), self.kind)
                                if p is not None:
                                    code = p[0][place(p[1])]
                                    if not scales[t] == scale:
                                        ratio = np.float32(scales[t] / scale) if scale > 0 else np.float32(0)
                                        code = encode(value(code, self.kind).astype(np.float32) * ratio, self.kind)
                                rec[place(t)] = code
                            f[which] = scale
                        for t, p in enumerate(part):
                            f[16 + t] = old.floats(p[0])[16 + p[1]] if p is not None else 0.0
        return kept

    def read(self, starts, lengths, tables, layer, layers, max_tokens, fill):
        """k, v and weights as the read call leaves buffers filled with `fill`."""
        n = len(lengths)
        k = np.full((layers, n, max_tokens, self.kvh, self.d), fill, dtype=np.float32)
        v = k.copy()
        w = np.full((layers, n, max_tokens, self.kvh), fill, dtype=np.float32)
        for l in range(layers):
            for i in range(n):
                for j in range(min(lengths[i], max_tokens)):
                    for g in range(self.kvh):
                        at = self.slot(tables[i], layer + l, g, (starts[i] if starts else 0) + j)
                        if at is None:
                            continue
                        f = self.floats(at[0])
                        k[l, i, j, g] = value(at[0][self.k_at(at[1])], self.kind).astype(np.float32) * f[0]
                        v[l, i, j, g] = value(at[0][self.v_at(at[1])], self.kind).astype(np.float32) * f[1]
                        w[l, i, j, g] = f[16 + at[1]]
        return k.reshape(layers, n, max_tokens, -1), v.reshape(layers, n, max_tokens, -1), w


def page_tables(rng, lengths, page_tokens, max_pages, pool_pages, first_page=0):
    """Scattered pages for sequences of these lengths, -1 behind them."""
    order = list(first_page + rng.permutation(pool_pages - first_page))
    out = np.full((len(lengths), max_pages), -1, dtype=np.int32)
    for i, n in enumerate(lengths):
        for p in range(-(-n // page_tokens)):
            out[i, p] = order.pop()
    return out
