"""Rotary positions, a paged cache and attention against it in numpy, from their definitions, in 64
bits; and batches of sequences laid out at random over a cache whose unused parts hold NaN."""
from __future__ import annotations

import numpy as np

import f8_reference as f8
import mensurflow_amd as mf

EPS32 = 2.0 ** -24    # half a step of fp32, relative
ANGLE = 1e-7          # what a cosine or sine may be off, with 2.5e-16 of the angle
HELD = {"f32": np.float32, "bf16": np.uint16, "e4m3": np.uint8}
BAD = (-1, 1 << 20, np.iinfo(np.int32).max, np.iinfo(np.int32).min)  # page numbers that no cache has


def dev(x, stream, dtype=None):
    return mf.DeviceArray.from_numpy(np.ascontiguousarray(x, dtype), stream)


# ---- rotation -------------------------------------------------------------------------------------


def steps(rot, base=10000.0, factor=1.0, original=0.0, slow=1.0, fast=32.0):
    step = base ** (-2 * np.arange(rot // 2) / max(rot, 1))
    kept = np.zeros(rot // 2)
    if original:
        kept = np.clip((original * step / (2 * np.pi) - slow) / (fast - slow), 0, 1)
    return step * (kept + (1 - kept) / factor)


def turn(x, positions, step, layout, amplitude=1.0, backward=False):
    """(x turned, how far fp32 may be from it): x [rows, heads, d]."""
    x = np.asarray(x, np.float64)
    half = len(step)
    out, off = x.copy(), np.zeros_like(x)
    w = np.asarray(positions, np.float64)[:, None, None] * step
    cos, sin = np.cos(w), np.sin(w) * (-1 if backward else 1)
    first = slice(0, half) if layout == mf.ROTARY_HALVES else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if layout == mf.ROTARY_HALVES else slice(1, 2 * half, 2)
    a, b = x[..., first], x[..., second]
    out[..., first] = amplitude * (a * cos - b * sin)
    out[..., second] = amplitude * (b * cos + a * sin)
    # The cosine's and sine's own error, their product with the amplitude, and two products and a sum.
    bound = abs(amplitude) * (np.abs(a) + np.abs(b)) * (ANGLE + 2.5e-16 * np.abs(w) + 4 * EPS32)
    off[..., first], off[..., second] = bound, bound
    return out, off


# ---- a cache's numbers ----------------------------------------------------------------------------


def bf16_bits(x):
    """fp32 to the bits of bf16, to nearest, ties to even; NaN stays NaN."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    bits = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), bits)


def bf16_values(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32)


def rows_to_held(x, held):
    """(numbers, scales) of rows x [..., d] as a cache holds them; scales None but in 8 bits."""
    x = np.asarray(x, np.float32)
    if held == "f32":
        return x, None
    if held == "bf16":
        return bf16_bits(x), None
    codes, scales = f8.quantize(x.reshape(-1, x.shape[-1]))
    return codes.reshape(x.shape), scales[:, 0].reshape(x.shape[:-1])


def held_to_rows(numbers, scales):
    """What the numbers of a cache stand for, in 64 bits."""
    if numbers.dtype == np.float32:
        return numbers.astype(np.float64)
    if numbers.dtype == np.uint16:
        return bf16_values(numbers).astype(np.float64)
    return f8.VALUES[numbers] * scales.astype(np.float64)[..., None]


# ---- batches --------------------------------------------------------------------------------------


class Paged:
    """A batch over a cache: counts [(rows, tokens)] of each sequence, rows in front of the first and
    behind the last, a shared prefix. Pages lie at random; every number that belongs to no token is
    NaN (in 8 bits NaN codes under NaN scales), and entries of the tables that no token uses name pages
    that there are not."""

    def __init__(self, rng, stream, counts, heads, d, held, page=16, prefix=0, layout="heads",
                 front=0, behind=0, even=False, spare=2, width=None, spread=1.0):
        self.stream, self.heads, self.d, self.held, self.page = stream, heads, d, held, page
        self.counts, self.prefix, self.layout = list(counts), prefix, layout
        used = [-(-max(t, 0) // page) for _, t in counts]
        self.width = max(used + [1]) if width is None else width
        shared = -(-prefix // page)
        self.pages = sum(used) + shared + spare
        order = rng.permutation(self.pages)
        self.table = np.array(BAD, np.int32)[rng.integers(0, len(BAD), (len(counts), self.width))]
        at = shared
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.prefix_pages = order[:shared].astype(np.int32)
        self.starts = front + np.concatenate(([0], np.cumsum([n for n, _ in counts]))).astype(np.int32)
        self.rows = int(self.starts[-1]) + behind
        self.lengths = np.array([t for _, t in counts], np.int32)
        self.even = even
        # The cache, [pages, heads, page, d].
        self.k, self.ks = self._empty()
        self.v, self.vs = self._empty()
        self.size = np.exp(spread * 0.4 * rng.standard_normal(d))

        def fill(numbers, scales, x, pages, tokens):
            values, s = rows_to_held(x, held)
            for t in range(tokens):
                numbers[pages[t // page], :, t % page] = values[t]
                if scales is not None:
                    scales[pages[t // page], :, t % page] = s[t]

        self.fill = fill
        for s, (_, tokens) in enumerate(counts):
            for numbers, scales, size in ((self.k, self.ks, self.size), (self.v, self.vs, 1.0)):
                fill(numbers, scales, rng.standard_normal((max(tokens, 0), heads, d)) * size,
                     self.table[s], tokens)
        for numbers, scales, size in ((self.k, self.ks, self.size), (self.v, self.vs, 1.0)):
            fill(numbers, scales, rng.standard_normal((prefix, heads, d)) * size, self.prefix_pages,
                 prefix)

    def _empty(self):
        shape = (self.pages, self.heads, self.page, self.d)
        if self.held == "f32":
            return np.full(shape, np.nan, np.float32), None
        if self.held == "bf16":
            return np.full(shape, 0x7FC0, np.uint16), None
        return np.full(shape, 0x7F, np.uint8), np.full(shape[:3], np.nan, np.float32)

    def _upload(self, x):
        if self.layout == "heads":
            return dev(x, self.stream)
        if self.layout == "tokens":     # [pages, page, heads, d]
            return dev(x.transpose(0, 2, 1, 3), self.stream).transpose(1, 2)
        # Rows 16 bytes apart from one another, pages in the second dimension.
        unit = 16 // x.dtype.itemsize
        wide = np.zeros((x.shape[1], x.shape[0], x.shape[2], x.shape[3] + unit), x.dtype)
        wide[..., :x.shape[3]] = x.transpose(1, 0, 2, 3)
        return dev(wide, self.stream).slice(3, 0, x.shape[3]).transpose(0, 1)

    def cache(self):
        self.dk, self.dv = self._upload(self.k), self._upload(self.v)
        if self.held != "e4m3":
            return mf.KvCache(self.dk, self.dv)
        self.dks, self.dvs = dev(self.ks, self.stream), dev(self.vs, self.stream)
        return mf.KvCache(self.dk, self.dv, self.dks, self.dvs)

    def batch(self):
        return mf.KvBatch(dev(self.lengths, self.stream), dev(self.table, self.stream),
                          starts=None if self.even else dev(self.starts, self.stream),
                          prefix=self.prefix,
                          prefix_pages=dev(self.prefix_pages, self.stream) if self.prefix else None)

    def tokens_of(self, s):
        """(keys, values) of sequence s in 64 bits, the prefix in front: [tokens, heads, d]."""
        out = []
        for numbers, scales in ((self.k, self.ks), (self.v, self.vs)):
            rows = []
            for pages, count in ((self.prefix_pages, self.prefix),
                                 (self.table[s], max(int(self.lengths[s]), 0))):
                t = np.arange(count)
                at, off = pages[t // self.page] if count else t, t % self.page
                rows.append(held_to_rows(numbers[at, :, off],
                                         None if scales is None else scales[at, :, off]))
            out.append(np.concatenate(rows))
        return out

    def attend(self, q, scale=None, causal=True, absent=()):
        """(out, bound) for q [rows, q_heads, d]: out NaN at rows of no sequence, bound what fp32
        sums in any order may be off. `absent`: (sequence, token) pairs that count as absent."""
        q = np.asarray(q, np.float64)
        group = q.shape[1] // self.heads
        scale = float(np.float32(1 / np.sqrt(self.d))) if scale is None else float(np.float32(scale))
        out, bound = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
        for s, (n, tokens) in enumerate(self.counts):
            k, v = self.tokens_of(s)
            keep = np.ones(len(k), bool)
            for seq, t in absent:
                if seq == s:
                    keep[self.prefix + t] = False
            for i in range(n):
                row = self.starts[s] + i
                seen = self.prefix + (max(0, min(tokens, tokens - n + i + 1)) if causal else tokens)
                at = np.flatnonzero(keep[:seen])
                for h in range(q.shape[1]):
                    kk, vv = k[at, h // group], v[at, h // group]
                    x = q[row, h]
                    score = scale * (kk @ x)
                    if not len(at):
                        out[row, h], bound[row, h] = 0, 0
                        continue
                    p = np.exp(score - score.max())
                    p /= p.sum()
                    out[row, h] = p @ vv
                    # A score: its d products' and sums' roundings, its scales', and the exponent's own
                    # in base 2, twice (its own and the maximum's); sums of as many terms as tokens.
                    wide = abs(scale) * (np.abs(kk) @ np.abs(x))
                    off = 2 * EPS32 * ((self.d + 8) * wide.max() + 4)
                    bound[row, h] = (np.expm1(2 * off) + (2 * len(at) + 16) * EPS32) * (
                        p @ np.abs(vv)) + 1e-37
        return out, bound


def attention_error(got, want):
    """The 2-norm of the difference over that of the result, over rows that have one."""
    there = ~np.isnan(want)
    d = got.astype(np.float64)[there] - want[there]
    return float(np.linalg.norm(d) / max(np.linalg.norm(want[there]), 1e-300))
