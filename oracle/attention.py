"""64-bit restatement of attention over packed prompts, of the 4-bit cache and of token log probabilities -- TEST
INFRASTRUCTURE ONLY. Plain numpy loops over rows and heads, written from the formulas the header states.
"""
from __future__ import annotations

import math

import numpy as np

GROUP = 32
f64 = np.float64


def attend_row(q, k, v, pos, scale, causal=True, window=0):
    """One query row over one kv head: (y, sum w |v|, largest error a score can have per unit of rounding).

    ``k`` / ``v`` [keys, dim]; the second result weighs what rounding a weight costs, the third is |scale| sum |q| |k| over the
    channels, at the key where that is largest."""
    keys = k.shape[0]
    last = min(pos, keys - 1) if causal else keys - 1
    first = max(0, pos - window + 1) if window > 0 else 0
    dim = v.shape[1]
    if last < first:
        return np.zeros(dim), np.zeros(dim), 0.0
    q, k, v = q.astype(f64), k[first:last + 1].astype(f64), v[first:last + 1].astype(f64)
    s = scale * (k @ q)
    with np.errstate(invalid="ignore"):
        w = np.exp(s - s.max())
        w /= w.sum()
        size = abs(scale) * float(np.max(np.abs(k) @ np.abs(q)))
        return w @ v, w @ np.abs(v), size


def prompt(q, k, v, q_lengths, k_lengths, causal=True, window=0, scale=None):
    """Packed rows: (y [rows, heads, dim], sum w |v| of the same shape, score sizes [rows, heads, 1])."""
    heads, group = q.shape[1], q.shape[1] // k.shape[1]
    scale = scale or 1.0 / math.sqrt(q.shape[2])
    y, weight, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((q.shape[0], heads, 1))
    q0 = k0 = 0
    for nq, nk in zip(q_lengths, k_lengths):
        for i in range(nq):
            for h in range(heads):
                y[q0 + i, h], weight[q0 + i, h], size[q0 + i, h] = attend_row(
                    q[q0 + i, h], k[k0:k0 + nk, h // group], v[k0:k0 + nk, h // group], nk - nq + i, scale, causal, window)
        q0, k0 = q0 + nq, k0 + nk
    return y, weight, size


def rotary(x, positions, frequencies, norm=None, eps=1e-6, interleaved=False, amplitude=1.0):
    """[rows, heads, dim] normed (``norm`` [dim] or None) and turned: (y, the sizes |x^_a cos| + |x^_b sin| of its two products), in 64 bits."""
    y = x.astype(f64)
    if norm is not None:
        y = y / np.sqrt(np.mean(y * y, -1, keepdims=True) + f64(np.float32(eps))) * norm.astype(f64)
    size = np.abs(y)
    n = len(frequencies)
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        t = positions.astype(f64) * f64(frequencies[i])
        c, s = (f64(np.float32(amplitude)) * f(t)[:, None] for f in (np.cos, np.sin))
        p, q = y[..., a].copy(), y[..., b].copy()
        y[..., a], y[..., b] = p * c - q * s, q * c + p * s
        size[..., a], size[..., b] = abs(p * c) + abs(q * s), abs(q * c) + abs(p * s)
    return y, size


def quantize(x):
    """[..., dim] as (codes, scale f16, lowest f16), groups of 32 channels, every decision in 64 bits."""
    g = np.clip(x.astype(f64), -65408, 65408).reshape(x.shape[:-1] + (-1, GROUP))
    lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    scale, lowest = ((hi - lo) / 15.0).astype(np.float32).astype(np.float16), lo.astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        steps = (g - lowest.astype(f64)) / scale.astype(f64)
    code = np.clip(np.rint(np.where(scale > 0, steps, 0.0)), 0, 15).astype(np.uint8)
    return code, scale, lowest


def values(code, scale, lowest):
    """What codes stand for: f16, rounded once."""
    v = lowest.astype(f64) + code.astype(f64) * scale.astype(f64)
    return v.astype(np.float16).reshape(v.shape[:-2] + (-1,))


class Cache:
    """The pages as plain arrays in the layout of the header."""

    def __init__(self, n_pages, page_size, n_kv, dim, table):
        self.page, self.table = page_size, np.asarray(table)
        shape = (n_pages, n_kv, page_size)
        self.codes = [np.zeros(shape + (dim // 2,), np.uint8) for _ in range(2)]
        self.params = [np.zeros(shape + (dim // GROUP, 2), np.float16) for _ in range(2)]

    def place(self, s, t):
        if t < 0 or t // self.page >= self.table.shape[1]:
            return None
        p = self.table[s, t // self.page]
        return (int(p), t % self.page) if 0 <= p < self.codes[0].shape[0] else None

    def store(self, s, t, rows):
        """rows: the (key, value) row [n_kv, dim] of position t."""
        at = self.place(s, t)
        if at is None:
            return
        for x, codes, params in zip(rows, self.codes, self.params):
            code, scale, lowest = quantize(x)
            flat = code.reshape(code.shape[0], -1)
            codes[at[0], :, at[1]] = flat[:, 0::2] | (flat[:, 1::2] << 4)
            p = np.concatenate([scale, lowest], -1)
            p[np.isnan(x.astype(f64)).reshape(code.shape).any(-1)] = np.nan
            params[at[0], :, at[1]] = p

    def load(self, which, s, t):
        """Position t's row [n_kv, dim] as f16, zeros where there is no page."""
        at = self.place(s, t)
        codes, params = self.codes[which], self.params[which]
        if at is None:
            return np.zeros((codes.shape[1], codes.shape[3] * 2), np.float16)
        c, p = codes[at[0], :, at[1]], params[at[0], :, at[1]]
        code = np.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1, GROUP)
        return values(code, p[..., :1], p[..., 1:])

    def attention(self, q, lengths, tokens, window=0, scale=None):
        heads, n_kv = q.shape[1], self.codes[0].shape[1]
        scale = scale or 1.0 / math.sqrt(q.shape[2])
        y, weight, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2] + (1,))
        for s, n in enumerate(lengths):
            n = max(0, int(n))
            for i in range(tokens):
                pos = n - tokens + i
                first = max(0, pos - window + 1) if window else 0
                seen = [t for t in range(first, min(pos + 1, self.table.shape[1] * self.page)) if self.place(s, t) is not None]
                if not seen:
                    continue
                k, v = (np.stack([self.load(w, s, t) for t in seen], 1) for w in (0, 1))
                for h in range(heads):
                    g = h // (heads // n_kv)
                    r = s * tokens + i
                    y[r, h], weight[r, h], size[r, h] = attend_row(q[r, h], k[g], v[g], len(seen) - 1, scale)
        return y, weight, size


    def prompt_attention(self, q, starts, lengths, window=0, sinks=0, scale=None):
        """Packed rows: (y, sum w |v|, score sizes, largest |v| seen [rows, heads, 1]); rows of no sequence are NaN."""
        heads, n_kv = q.shape[1], self.codes[0].shape[1]
        scale = scale or 1.0 / math.sqrt(q.shape[2])
        y, weight = np.full(q.shape, np.nan), np.zeros(q.shape)
        size, most = np.zeros(q.shape[:2] + (1,)), np.zeros(q.shape[:2] + (1,))
        for s, length in enumerate(lengths):
            length, first, end = max(0, int(length)), max(0, int(starts[s])), min(q.shape[0], int(starts[s + 1]))
            held = [t for t in range(min(length, self.table.shape[1] * self.page)) if self.place(s, t) is not None] if first < end else []
            k, v = (np.stack([self.load(w, s, t) for t in held], 1) if held else None for w in (0, 1))
            held = np.array(held, np.int64)
            for r in range(first, end):
                pos = length - end + r
                see = (held <= pos) & ((held > pos - window) | (held < sinks) if window else True)
                y[r] = 0
                if not see.any():
                    continue
                for h in range(heads):
                    g = h // (heads // n_kv)
                    y[r, h], weight[r, h], size[r, h] = attend_row(q[r, h], k[g][see], v[g][see], int(see.sum()) - 1, scale)
                    most[r, h] = np.abs(v[g][see].astype(f64)).max()
        return y, weight, size, most


def token_logprobs(x, tokens, top):
    """(logprob, entropy, ids, logprobs of the best) in 64 bits."""
    rows, vocab = x.shape
    out = [np.zeros(rows), np.zeros(rows), np.full((rows, top), -1, np.int32), np.full((rows, top), np.nan)]
    for r in range(rows):
        v = x[r].astype(f64)
        m = v.max()   # NaN if there is one
        with np.errstate(invalid="ignore", divide="ignore"):
            e = np.exp(v - m)
            lse = m + np.log(e.sum())
            p = e / e.sum()
            out[1][r] = lse - np.sum(np.where(p > 0, p * np.where(p > 0, v, 0.0), 0.0)) if np.isfinite(m) else np.nan
            t = int(tokens[r])
            out[0][r] = 0.0 if t == -1 else v[t] - lse if 0 <= t < vocab else np.nan
            ids = [i for i in np.argsort(np.where(np.isnan(v), np.inf, -v), kind="stable") if not np.isnan(v[i])][:top]
            out[2][r, :len(ids)] = ids
            out[3][r, :len(ids)] = v[ids] - lse
    return tuple(out)
