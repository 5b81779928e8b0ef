"""The 8-bit KV cache in plain 64-bit Python: what lastro_kv8_* must leave behind, block by block."""
import math

import numpy as np

PAGE, BLOCK = 64, 16
QMAX = {"e4m3": 448.0, "int8": 127.0}


def scale_for(amax: float, fmt: str) -> float:
    """The smallest power of two 2^e, e >= -126, with amax <= qmax * 2^e; NaN when amax is not finite."""
    if not math.isfinite(amax):
        return math.nan
    e = -126
    while amax > QMAX[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def quantise(x: np.ndarray, fmt: str) -> np.ndarray:
    """Nearest code values (as f64) to x, ties to even; |x| <= qmax."""
    if fmt == "int8":
        return np.rint(x)
    _, e = np.frexp(np.maximum(np.abs(x), 2.0 ** -6))  # 3 fraction bits below the leading one; 2^-9 steps below 2^-6
    step = np.exp2(e - 4.0)
    return np.rint(x / step) * step


def need(x: np.ndarray, fmt: str) -> float:
    if x.size == 0:
        return 2.0 ** -126
    a = np.abs(x)
    return scale_for(math.nan if not np.isfinite(a).all() else float(a.max()), fmt)


class Side:
    """K or V of one sequence and head: rows of code values and one scale per block."""

    def __init__(self, d, fmt):
        self.d, self.fmt, self.codes, self.scales = d, fmt, np.zeros((0, d)), []

    def append(self, rows):
        at, end = self.codes.shape[0], self.codes.shape[0] + rows.shape[0]
        self.codes = np.concatenate([self.codes, np.zeros_like(rows)])
        for blk in range(at // BLOCK, -(-end // BLOCK)):
            lo, hi = max(at, blk * BLOCK), min(end, (blk + 1) * BLOCK)
            if hi <= lo:
                continue
            new = rows[lo - at:hi - at]
            s = need(new, self.fmt)
            if lo > blk * BLOCK:  # earlier rows in the block
                was = self.scales[blk]
                s = math.nan if math.isnan(s) or math.isnan(was) else max(s, was)
                if not math.isnan(s) and s != was:
                    self.codes[blk * BLOCK:lo] = quantise(self.codes[blk * BLOCK:lo] * (was / s), self.fmt)
                self.scales[blk] = s
            else:
                self.scales.append(s)
            self.codes[lo:hi] = quantise(new / s, self.fmt) if not math.isnan(s) else 0.0

    def values(self):
        n = self.codes.shape[0]
        s = np.repeat(np.array(self.scales + [0.0]), BLOCK)[:n] if n else np.zeros(0)
        return self.codes * s[:, None]

    def gather(self, keep):
        out = Side(self.d, self.fmt)
        v = self.values()[keep]
        for lo in range(0, len(keep), BLOCK):
            out.append(v[lo:lo + BLOCK])
        return out


class Cache:
    """Every sequence and head: side[b][h] = {"k": Side, "v": Side}."""

    def __init__(self, n_seqs, kv_heads, d, fmt):
        self.d, self.fmt, self.kv_heads = d, fmt, kv_heads
        self.side = [[{w: Side(d, fmt) for w in "kv"} for _ in range(kv_heads)] for _ in range(n_seqs)]

    def length(self, b):
        return self.side[b][0]["k"].codes.shape[0]

    def append(self, b, k, v):
        """k, v [n, kv_heads, d] f64"""
        for h, s in enumerate(self.side[b]):
            s["k"].append(k[:, h])
            s["v"].append(v[:, h])

    def attend(self, b, q, scale):
        """q [n, heads, d] -> out [n, heads, d], weights each slot received [kv_heads, len], and the largest
        sum_j |q_j k_j| * scale of a score, which its rounding errors are proportional to"""
        n, heads, _ = q.shape
        length, G = self.length(b), heads // self.kv_heads
        out, mass, big = np.zeros_like(q), np.zeros((self.kv_heads, length)), 0.0
        for h in range(self.kv_heads):
            k, v = self.side[b][h]["k"].values(), self.side[b][h]["v"].values()
            for i in range(n):
                see = max(0, length - n + i + 1)
                if see == 0:
                    continue
                for g in range(G):
                    x = q[i, h * G + g]
                    s = scale * (k[:see] @ x)
                    big = max(big, float(abs(scale) * (np.abs(k[:see]) @ np.abs(x)).max()))
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[i, h * G + g] = p @ v[:see]
                    mass[h, :see] += p
        return out, mass, big

    def evict(self, b, mass, budget, recent):
        """mass [kv_heads, len] -> kept slots per head; the sequence becomes the kept rows"""
        length, kept = self.length(b), []
        for h in range(self.kv_heads):
            if length <= budget:
                keep = np.arange(length)
            else:
                cand = length - recent
                key = np.where(np.isnan(mass[h, :cand]), np.inf, mass[h, :cand])
                order = sorted(range(cand), key=lambda t: (not np.isnan(mass[h, t]), -key[t], t))
                keep = np.array(sorted(order[:budget - recent]) + list(range(cand, length)), dtype=int)
            kept.append(keep)
            for w in "kv":
                self.side[b][h][w] = self.side[b][h][w].gather(keep)
        return kept
