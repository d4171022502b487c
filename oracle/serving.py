"""Plain NumPy forms, in 64 bits, of the operators that a decoder serves with:
the 4-bit key/value cache, attention over it, and log probabilities by token
id.  Written from the formulas; loops where they are clearest."""

from __future__ import annotations

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
GROUP = 32


def quantise(x):
    """Codes (..., D/2) and scale bytes (..., D/32), uint8, of float32 x (..., D)."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP).astype(np.float64)
    amax = np.abs(g).max(-1)
    held = amax < 2.0 ** 127  # false for NaN
    safe = np.where(held & (amax > 0), amax, 6.0)
    e = np.maximum(np.ceil(np.log2(safe / 6)), -119)
    byte = np.where(held, np.where(amax > 0, e + 127, 127), 255).astype(np.uint8)
    y = np.abs(np.where(held[..., None], g, 0)) * 2.0 ** -e[..., None]
    off = np.abs(y[..., None] - E2M1)
    near = off == off.min(-1, keepdims=True)
    # Of two as near, the even code (neighbours are never both even).
    code = np.argmax(near * np.where(np.arange(8) % 2 == 0, 2, 1), -1)
    code = np.where(held[..., None], code | (np.signbit(g) * 8), 0).astype(np.uint8).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def values(codes, scales):
    """float64 (..., D) that codes and scale bytes stand for."""
    n = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    size = E2M1[n & 7] * np.where(n & 8, -1.0, 1.0)
    scale = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return size * np.repeat(scale, GROUP, -1)


class Cache:
    """The arrays of a cache and its page table, in host memory."""

    def __init__(self, pages, heads, page_size, D, table):
        self.page_size, self.heads, self.D, self.pages = page_size, heads, D, pages
        self.table = np.asarray(table, np.int32)
        shape = (pages, heads, page_size)
        self.codes = [np.zeros((*shape, D // 2), np.uint8) for _ in range(2)]
        self.scales = [np.zeros((*shape, D // GROUP), np.uint8) for _ in range(2)]

    def slot(self, b, pos):
        """(page, token of the page) of a sequence's token, or None."""
        if not 0 <= pos < self.table.shape[1] * self.page_size:
            return None
        page = int(self.table[b, pos // self.page_size])
        return (page, pos % self.page_size) if 0 <= page < self.pages else None

    def write(self, k, v, start=None, count=None):
        """k, v (B, T, heads, D); returns where each sequence's next call starts."""
        B, T = k.shape[:2]
        start, count = spans(B, T, start, count)
        for i, x in enumerate((k, v)):
            codes, scales = quantise(x)
            for b in range(B):
                for t in range(count[b]):
                    at = self.slot(b, start[b] + t)
                    if at:
                        self.codes[i][at[0], :, at[1]], self.scales[i][at[0], :, at[1]] = codes[b, t], scales[b, t]
        return start + count

    def token(self, i, b, pos):
        """float64 (heads, D) of a token's keys (i = 0) or values (1), or None."""
        at = self.slot(b, pos)
        return None if at is None else values(self.codes[i][at[0], :, at[1]], self.scales[i][at[0], :, at[1]])

    def read(self, T, start=None, count=None):
        B = self.table.shape[0]
        start, count = spans(B, T, start, count)
        out = np.zeros((2, B, T, self.heads, self.D))
        for i in range(2):
            for b in range(B):
                for t in range(count[b]):
                    x = self.token(i, b, start[b] + t)
                    if x is not None:
                        out[i, b, t] = x
        return out[0], out[1]

    def attention(self, q, causal, scale, start=None, count=None):
        """o (B, T, Hq, D), lse (B, Hq, T), and for error bounds the sum of
        p |v| (like o) and the largest sum of |q k| scale of a row (like lse)."""
        B, T, Hq, D = q.shape
        start, count = spans(B, T, start, count)
        q = q.astype(np.float64)
        o, lse = np.zeros(q.shape), np.full((B, Hq, T), -np.inf)
        weight, reach = np.zeros(q.shape), np.zeros((B, Hq, T))
        for b in range(B):
            known = [(j, self.token(0, b, j), self.token(1, b, j)) for j in range(max(0, start[b] + count[b]))]
            known = [(j, k, v) for j, k, v in known if k is not None]
            if not known:
                continue
            at = np.array([j for j, _, _ in known])
            ks, vs = (np.stack([x[n] for x in known]) for n in (1, 2))
            for h in range(Hq):
                k, v = ks[:, h // (Hq // self.heads)], vs[:, h // (Hq // self.heads)]
                for t in range(count[b]):
                    see = at <= start[b] + t if causal else np.ones(len(at), bool)
                    if not see.any():
                        continue
                    s = k[see] @ q[b, t, h] * scale
                    m = s.max()
                    e = np.exp(s - m)
                    lse[b, h, t] = m + np.log(e.sum())
                    o[b, t, h] = e @ v[see] / e.sum()
                    weight[b, t, h] = e @ np.abs(v[see]) / e.sum()
                    reach[b, h, t] = (np.abs(k[see]) @ np.abs(q[b, t, h])).max() * scale
        return o, lse, weight, reach


def spans(B, T, start, count):
    start = np.zeros(B, np.int64) if start is None else np.asarray(start, np.int64)
    count = np.full(B, T, np.int64) if count is None else np.clip(np.asarray(count, np.int64), 0, T)
    return start, count


def token_logprobs(x, tokens, top):
    """logp, lse, entropy, top ids and their log probabilities of rows x, float64."""
    x = np.asarray(x, np.float64)
    rows, classes = x.shape
    m = x.max(-1, keepdims=True)
    logs = np.log(np.exp(x - m).sum(-1, keepdims=True))
    lse = (m + logs)[:, 0]
    logp = (x - m) - logs  # not x - lse: a far m swallows ln s even here
    p = np.exp(logp)
    entropy = -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(-1)
    known = (tokens >= 0) & (tokens < classes)
    chosen = np.where(known, logp[np.arange(rows), np.clip(tokens, 0, classes - 1)], 0)
    order = np.argsort(-x, -1, kind="stable")[:, :top]
    return chosen, lse, entropy, order, np.take_along_axis(logp, order, -1)


def token_logprobs_bwd(x, tokens, d_logp, d_entropy):
    """Gradient of sum(d_logp * logp + d_entropy * entropy), float64."""
    x = np.asarray(x, np.float64)
    rows, classes = x.shape
    _, lse, entropy, _, _ = token_logprobs(x, tokens, 1)
    logp = x - lse[:, None]
    p = np.exp(logp)
    known = (tokens >= 0) & (tokens < classes)
    d = np.where(known, d_logp, 0)
    plogp = np.where(p > 0, p * np.where(p > 0, logp, 0), 0)
    grad = -p * d[:, None] - d_entropy[:, None] * (plogp + p * entropy[:, None])
    grad[np.arange(rows)[known], tokens[known]] += d[known]
    return grad
