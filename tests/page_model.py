"""Plain model of the page cache and of rotary positions, for the tests: NumPy, values in 64 bits, written from the
definitions in include/mmreshard.h and from nothing of the library."""
from __future__ import annotations

import numpy as np

TAU = np.longdouble(2) * np.longdouble("3.14159265358979323846264338327950288")
EPS = {"F32": 2.0 ** -23, "BF16": 2.0 ** -7, "F16": 2.0 ** -10}  # a rounding is off by half of it at most


def to_bits(x, type):
    """Values -> raw bits of the type, rounded to nearest even."""
    x = np.asarray(x, dtype=np.float32)
    if type == "F32":
        return x.view(np.uint32)
    if type == "F16":
        return x.astype(np.float16).view(np.uint16)
    u = x.view(np.uint32)
    return ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)


def from_bits(b, type):
    """Raw bits -> values in 64 bits."""
    if type == "F32":
        return b.view(np.float32).astype(np.float64)
    if type == "F16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << np.uint32(16)).view(np.float32).astype(np.float64)


RAW = {"F32": np.uint32, "BF16": np.uint16, "F16": np.uint16, "U8": np.uint8, "S8": np.uint8, "F8E4M3FN": np.uint8, "F64": np.uint64}


class Cache:
    """pools: arrays [pages, ...] of raw bits, whole (all heads)."""

    def __init__(self, S, B, P, T, pools):
        self.S, self.B, self.P, self.T = S, B, P, T
        self.table = np.zeros((S, B), dtype=np.int32)
        self.lengths = np.zeros(S, dtype=np.int32)
        self.refs = np.zeros(P, dtype=np.int32)
        self.pools = pools

    def blocks(self, tokens):
        return -(-int(tokens) // self.T)

    def free_pages(self):
        return np.flatnonzero(self.refs == 0)

    def extend(self, seqs, counts):
        need = sum(self.blocks(self.lengths[s] + c) - self.blocks(self.lengths[s]) for s, c in zip(seqs, counts))
        f = list(self.free_pages())
        assert need <= len(f)
        for s, c in zip(seqs, counts):
            for b in range(self.blocks(self.lengths[s]), self.blocks(self.lengths[s] + c)):
                self.table[s, b] = f.pop(0)
                self.refs[self.table[s, b]] = 1
            self.lengths[s] += c

    def fork(self, parents, children):
        f = list(self.free_pages())
        for p, c in zip(parents, children):
            full = self.lengths[p] // self.T
            self.table[c, :full] = self.table[p, :full]
            np.add.at(self.refs, self.table[p, :full], 1)
            if self.lengths[p] % self.T:
                g = f.pop(0)
                for pool in self.pools:
                    pool[g] = pool[self.table[p, full]]
                self.table[c, full] = g
                self.refs[g] = 1
            self.lengths[c] = self.lengths[p]

    def free(self, seqs):
        for s in seqs:
            np.add.at(self.refs, self.table[s, :self.blocks(self.lengths[s])], -1)
            self.lengths[s] = 0

    def copy(self, src, dst):
        for pool in self.pools:
            pool[list(dst)] = pool[list(src)]

    def compact(self):
        live = int((self.refs != 0).sum())
        src = [p for p in range(live, self.P) if self.refs[p]]
        dst = [p for p in range(live) if not self.refs[p]]
        name = np.arange(self.P)
        name[src] = dst
        for pool in self.pools:
            pool[dst] = pool[src]
        self.refs[dst] = self.refs[src]
        self.refs[src] = 0
        for s in range(self.S):
            n = self.blocks(self.lengths[s])
            self.table[s, :n] = name[self.table[s, :n]]

    def places(self, seqs, begins):
        """{token: (position, page, row in the page)}"""
        out = {}
        for j, s in enumerate(seqs):
            for t in range(begins[j], begins[j + 1]):
                p = int(self.lengths[s]) - (begins[j + 1] - begins[j]) + (t - begins[j])
                out[t] = (p, int(self.table[s, p // self.T]), p % self.T)
        return out


def frequencies(rotary_dim, base=10000.0, scaling=None, factor=1.0, original_positions=0, low_turns=0.0, high_turns=0.0):
    """Radians per position, in the longest type there is."""
    i = np.arange(rotary_dim // 2, dtype=np.longdouble)
    f = np.longdouble(base) ** (-2 * i / rotary_dim)
    if scaling == "linear":
        return f / factor
    if scaling == "parts":
        w = np.clip((original_positions * f / TAU - low_turns) / np.longdouble(high_turns - low_turns), 0, 1)
        return f * w + f / factor * (1 - w)
    return f


def turn(x, positions, freq, interleaved=False, magnitude=1.0, backward=False):
    """x [..., dim] in 64 bits; positions broadcast over x's leading dims -> (result, |a| + |b| of every value's pair)."""
    half = len(freq)
    turns = np.asarray(positions, dtype=np.longdouble)[..., None] * (freq / TAU)
    angle = ((turns - np.floor(turns)) * TAU).astype(np.float64)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if backward else 1)
    y, size = np.array(x, dtype=np.float64), np.zeros(x.shape)
    first = (Ellipsis, slice(0, 2 * half, 2)) if interleaved else (Ellipsis, slice(0, half))
    second = (Ellipsis, slice(1, 2 * half, 2)) if interleaved else (Ellipsis, slice(half, 2 * half))
    a, b = x[first], x[second]
    y[first], y[second] = a * c - b * s, b * c + a * s
    size[first] = size[second] = np.abs(a) + np.abs(b)
    return y, size


def tolerance(want, size, type, magnitude=1.0):
    """Half a step of the type on the result, and in 32 bits before it: sine and cosine within 2^-23 (a rounding of the
    rest of a quarter turn, of the sum and of the factor), a product's rounding 2^-24, the sum's 2^-24 of the result; the
    products' bounds add up over the pair.  16-bit floats: below the normal range half a step is 2^-25 (F16)."""
    slack = magnitude * (2.0 ** -23 + 2.0 ** -24 + 2.0 ** -24) * size + 2.0 ** -24 * np.abs(want)
    return EPS[type] / 2 * np.abs(want) * (1 + 2.0 ** -20) + (1 + EPS[type]) * slack + (2.0 ** -25 if type == "F16" else 0.0)
