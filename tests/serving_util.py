"""Programs, batches and plain 64-bit forms of the rotary and paged cache operators."""
from __future__ import annotations

import numpy as np

from oracle import vmref
from pjrt_amd import graph as G
from pjrt_amd import vmprogram as V

U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # half a step, relative


def to_dt(x, dt):
    """Values as stored in dt (bf16 as its 16-bit patterns)."""
    if dt == "bf16":
        return vmref.f32_to_bf16(np.asarray(x, np.float32))
    return np.asarray(x).astype({"f32": np.float32, "f16": np.float16, "i8": np.int8}[dt])


def to_f64(x, dt):
    return (vmref.bf16_to_f32(x) if dt == "bf16" else np.asarray(x)).astype(np.float64)


class Case:
    """A batch over a paged cache: `seqs` of (new rows, length), random pages, and
    NaN in every slot of the pools that no position lies in."""

    def __init__(self, seqs, hq, hkv, hd, page, dt, cache=None, pad=0, window=0, seed=0, spare=3, max_pages=None,
                 first=0):
        self.rng = rng = np.random.default_rng(seed)
        self.seqs, self.hq, self.hkv, self.hd, self.page, self.dt = seqs, hq, hkv, hd, page, dt
        self.cache, self.window = cache or dt, window
        need = [-(-length // page) for _, length in seqs]
        self.MP = max_pages or max(1, max(need))
        self.N = sum(need) + spare
        order = rng.permutation(self.N).astype(np.int32)
        self.table = np.full((len(seqs), self.MP), -1, np.int32)
        self.cu = [first]
        at = 0
        for i, (n, length) in enumerate(seqs):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
            self.cu.append(self.cu[-1] + n)
        self.T = max(1, self.cu[-1] + pad)
        self.cu = np.asarray(self.cu, np.int32)
        self.lens = np.asarray([length for _, length in seqs], np.int32)
        shape = (self.N, hkv, page, hd)
        used = np.zeros((self.N, page), bool)
        for i, (_, length) in enumerate(seqs):
            for p in range(length):
                used[self.table[i, p // page], p % page] = True
        self.pools, self.scales = [], []
        for _ in range(2):
            if self.cache == "i8":
                self.pools.append(rng.integers(-127, 128, shape).astype(np.int8))
                s = rng.uniform(0.004, 0.02, shape[:3]).astype(np.float32)
                s[~used[:, None].repeat(hkv, 1)] = np.nan
                self.scales.append(s)
            else:
                x = rng.standard_normal(shape)
                x[~used[:, None].repeat(hkv, 1)] = np.nan
                self.pools.append(to_dt(x, self.cache))
        self.q = to_dt(rng.standard_normal((self.T, hq, hd)) * 1.5, dt)
        self.k = to_dt(rng.standard_normal((self.T, hkv, hd)), dt)
        self.v = to_dt(rng.standard_normal((self.T, hkv, hd)), dt)
        self.scale = hd ** -0.5

    def state(self):
        return [p.copy() for p in self.pools] + [s.copy() for s in self.scales]

    def batch(self):
        return [self.cu, self.lens, self.table]

    def declare(self, g):
        b = g.paged_batch(len(self.seqs), self.MP)
        return b, g.paged_cache(self.N, self.hkv, self.page, self.hd, self.cache)

    def attention_program(self):
        g = G.Graph()
        b, c = self.declare(g)
        q = g.input(self.q.shape, self.dt)
        g.output(g.paged_attention(q, c, b, self.scale, self.window))
        return g.build()

    def values(self, pool, i):
        """[length, hkv, hd] f64 of sequence i, NaN where its table has no page."""
        length = int(self.lens[i])
        p = np.arange(length)
        pages, slots = self.table[i][p // self.page], p % self.page
        ok = (pages >= 0) & (pages < self.N)
        pg = np.where(ok, pages, 0)
        x = to_f64(self.pools[pool], self.cache)[pg, :, slots] if self.cache != "i8" else \
            self.pools[pool][pg, :, slots].astype(np.float64) * self.scales[pool][pg, :, slots].astype(np.float64)[..., None]
        return x, ok

    def attention(self):
        """(out, sum of P |v|, largest |score|) in 64 bits."""
        q = to_f64(self.q, self.dt)
        out, mag, top = np.zeros(q.shape), np.zeros(q.shape), 0.0
        g = self.hq // self.hkv
        for i in range(len(self.seqs)):
            a, b = int(self.cu[i]), int(self.cu[i + 1])
            n, length = b - a, int(self.lens[i])
            if n <= 0 or length < n or length > self.MP * self.page:
                continue
            k, ok = self.values(0, i)
            v, _ = self.values(1, i)
            j, p = np.arange(length), np.arange(length - n, length)
            see = (j[None] <= p[:, None]) & ok[None]
            if self.window:
                see &= j[None] > p[:, None] - self.window
            for h in range(self.hq):
                kk, vv = np.where(ok[:, None], k[:, h // g], 0.0), np.where(ok[:, None], v[:, h // g], 0.0)
                s = np.where(see, q[a:b, h] @ kk.T * self.scale, -np.inf)
                top = max(top, float(np.abs(s[see]).max()) if see.any() else 0.0)
                m = s.max(-1, keepdims=True)
                e = np.exp(s - np.where(np.isfinite(m), m, 0.0))
                w = e / np.maximum(e.sum(-1, keepdims=True), 1e-300)
                out[a:b, h], mag[a:b, h] = w @ vv, w @ np.abs(vv)
        return out, mag, top

    def attention_tolerance(self, out, mag, top):
        """Per element: rounding P, the output's rounding, and f32 sums.  P is rounded to the
        queries' type, w (1 + d) with |d| <= half a step, and divided by the sum of the
        rounded ones: 2 half steps of sum w |v|.  Over i8 pages P times the value's scale is
        rounded to bf16 (f16 has no room for the scales' range; with f16 queries to the sum
        of two bf16 numbers, so |d| <= 2^-8 2^-8) and divided by the sum of the unrounded P:
        sum w (1 + d) v with |d| <= 2^-8 is off by at most 2^-8 sum w |v|.
        The sums: a score is off by at most (hd + 4) 2^-24 of sum |q k| scale, taken as 4
        times the largest score, which moves every weight by that factor; exp2, the
        sums and the division add at most 64 2^-24."""
        p = 0.0 if self.dt == "f32" else (U["bf16"] if self.dt == "bf16" else U["bf16"] ** 2) if self.cache == "i8" else U[self.dt]
        f32 = ((self.hd + 4) * 4 * top + 64 + 2 * top) * 2.0 ** -24
        return (2 * p + 2 * f32) * mag + U[self.dt] * np.abs(out) + 1e-30


def rotary_program(x_shape, dt, freq, norm, interleaved, magnitude=1.0, inverse=False, eps=1e-6, view=None):
    g = G.Graph()
    T, H, hd = x_shape
    src = g.input((T, H, hd) if view is None else view[0], dt)
    x = src if view is None else g.view(src, x_shape, view[1], view[2])
    pos = g.input((T,), "i32")
    w = g.input((hd,), "f32") if norm else None
    g.output(g.rotary(x, pos, freq, weight=w, eps=eps, interleaved=interleaved, magnitude=magnitude, inverse=inverse))
    return g.build()


def rotary_plain(x, pos, freq, interleaved, magnitude=1.0, inverse=False, weight=None, eps=1e-6):
    """(y, sum of |terms|) in 64 bits, by the two products of each pair."""
    x = np.asarray(x, np.float64)
    hd, R = x.shape[-1], len(freq)
    z = x if weight is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    turn = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float64)
    c, s = np.cos(turn)[:, None] * magnitude, np.sin(turn)[:, None] * magnitude * (-1.0 if inverse else 1.0)
    ia, ib = (np.arange(0, 2 * R, 2), np.arange(1, 2 * R, 2)) if interleaved else (np.arange(R), np.arange(R, 2 * R))
    y, mag = z.copy(), np.abs(z)
    y[..., ia], y[..., ib] = z[..., ia] * c - z[..., ib] * s, z[..., ib] * c + z[..., ia] * s
    mag[..., ia] = mag[..., ib] = (np.abs(z[..., ia]) + np.abs(z[..., ib])) * magnitude
    return y, mag
