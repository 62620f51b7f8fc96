"""Test support of the paged cache: random batches in pages, and what the operators give for them in 64 bits, written from
the definition (one row at a time over the positions that it sees)."""
from __future__ import annotations

import numpy as np

from kalosm_amd.fusor import PagedBatch, PagedKvCache, Tensor

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # of a rounding, relative to the value
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}  # the step below the normal range


def pack(a, dtype):
    """float64 / float32 values as the type's array (bf16: uint16 bit patterns), rounded to nearest even."""
    a = np.asarray(a, np.float32)
    if dtype == "f32":
        return a.copy()
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return a.astype(np.float16)
    u = np.ascontiguousarray(a).view(np.uint32)
    r = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def unpack(a, dtype):
    if dtype == "bf16":
        return (np.ascontiguousarray(a).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


class Pages:
    """A batch of ragged sequences: `new[i]` rows of sequence i, the last of its `lens[i]` positions, in pages in random order.
    Slots that hold no position of a sequence hold NaN.  `slot_major`: pages [page][slot][head]."""

    def __init__(self, seed, new, lens, hq, hkv, d, page, act, kept, slot_major=False, spare=2, before=0, behind=0, spread=1.0):
        rng = np.random.default_rng(seed)
        self.new, self.lens, self.hq, self.hkv, self.d, self.page, self.act, self.kept = new, lens, hq, hkv, d, page, act, kept
        self.slot_major, n = slot_major, len(new)
        need = [-(-x // page) for x in lens]
        self.cols = max(max(need), 1) + 1
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((n, self.cols), -1, np.int32)
        at = 0
        for i, c in enumerate(need):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.starts = (before + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        self.tokens = int(self.starts[-1]) + behind
        self.q = pack(spread * rng.standard_normal((self.tokens, hq, d)), act)
        shape = (self.pages, hkv, page, d)
        self.k, self.v = pack(rng.standard_normal(shape), kept), pack(rng.standard_normal(shape), kept)
        nan = pack(np.full((), np.nan), kept)
        used = np.zeros((self.pages, page), bool)
        for i, x in enumerate(lens):
            p = np.arange(x)
            used[self.table[i, p // page], p % page] = True
        for a in (self.k, self.v):
            a[(~used)[:, None, :, None] & np.ones(shape, bool)] = nan

    def put(self, dev):
        """The cache and the batch on the device."""
        def up(a):
            return Tensor.from_slice(dev, a.transpose(0, 2, 1, 3) if self.slot_major else a, self.kept)

        self.kt, self.vt = up(self.k), up(self.v)
        cache = PagedKvCache.over(Tensor(dev, self.k.shape, self.kept, ptr=self.kt.ptr), Tensor(dev, self.v.shape, self.kept, ptr=self.vt.ptr))
        if self.slot_major:
            cache._layers = [(self.kt.ptr, self.vt.ptr, self.hkv * self.page * self.d, self.d, self.hkv * self.d, self.pages, self.page)]
        batch = PagedBatch(Tensor.from_slice(dev, np.array(self.lens, np.int32), "i32"), Tensor.from_slice(dev, self.table, "i32"),
                           Tensor.from_slice(dev, self.starts, "i32"), tokens=self.tokens, max_new=max(self.new), max_len=max(self.lens))
        return cache, batch

    def held(self):
        """The pages as they are on the device now."""
        a = self.kt.as_slice(), self.vt.as_slice()
        return tuple(x.reshape(self.pages, self.page, self.hkv, self.d).transpose(0, 2, 1, 3) for x in a) if self.slot_major else a

    def rows(self):
        """(row, sequence, position) of every new row."""
        for i, m in enumerate(self.new):
            for r in range(m):
                yield int(self.starts[i]) + r, i, self.lens[i] - m + r

    def attention(self, scale, window=0):
        """The result in 64 bits, and how far each value may be off (attention_bound)."""
        q, k, v = unpack(self.q, self.act), unpack(self.k, self.kept), unpack(self.v, self.kept)
        out, bound = np.zeros((self.tokens, self.hq, self.d)), np.zeros((self.tokens, self.hq, self.d))
        g = self.hq // self.hkv
        for row, i, p in self.rows():
            j = np.arange(max(0, p - window + 1) if window else 0, min(p + 1, self.lens[i], self.cols * self.page))
            pages = self.table[i, j // self.page]
            j, pages = (x[(pages >= 0) & (pages < self.pages)] for x in (j, pages))
            if not len(j):
                continue
            ks, vs = k[pages, :, j % self.page], v[pages, :, j % self.page]  # [keys, hkv, d]
            for h in range(self.hkv):
                x = q[row, h * g:(h + 1) * g]
                s = scale * (x @ ks[:, h].T)
                w = np.exp(s - s.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                o = w @ vs[:, h]
                out[row, h * g:(h + 1) * g] = o
                size = scale * (np.abs(x) @ np.abs(ks[:, h]).T).max(1, keepdims=True)
                bound[row, h * g:(h + 1) * g] = attention_bound(o, w @ np.abs(vs[:, h]), np.abs(vs[:, h]).sum(0), size, len(j), self.d, self.act, self.kept)
        return out, bound


def attention_bound(o, mass, whole, size, keys, d, act, kept):
    """How far attention may be off: o the result, mass = sum w |v|, whole = sum |v|, size = the largest scale * sum |q| |k| of a key.

    A score is a sum of d products held in f32, in any order, of operands whose terms carry 2^-23 of the value (f32 operands go to
    the matrix cores in parts), scaled once and taken to base 2: off by at most ds = (d + 6) 2^-23 size.  Normalised weights are
    then off by a factor within exp(+-2 ds), and the exponential itself by 2^-21.  Each weight is rounded to the type of the pages
    where it is multiplied in 16 bits (half a step; f32 rows: in several terms, 2^-22).  Sums over the keys are f32: each of
    at most keys + 64 additions is off by 2^-24 of what has been summed, numerator and denominator alike.  The result is rounded once.

    Weights next to f16 values are f16 themselves, at 2^14 times their size relative to the largest (which is at most 1): where a term falls
    below f16's normal range its half step is 2^-25, that is 2^-39 of a weight of 1, whatever the weight's own size - a result to which the heavy
    positions contribute zeros can be off by that much of its small ones: 2^-39 sum |v| in all."""
    ds = (d + 6) * 2.0 ** -23 * size
    weight = HALF_STEP[kept] if act == kept and act != "f32" else 2.0 ** -22
    rel = np.expm1(2 * ds) + 2.0 ** -20 + weight + 2 * (keys + 64) * 2.0 ** -24
    inner = rel * mass + (2.0 ** -39 * whole if kept == "f16" else 0.0)
    return 1.01 * (HALF_STEP[act] * (np.abs(o) + inner) + inner) + SMALLEST[act]


def near(got, want, bound, what):
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.size} values off, first at {tuple(int(x) for x in np.argwhere(bad)[0])}: {got[bad][0]} for {want[bad][0]}, "
                           f"allowed {bound[bad][0]:.3g}; worst {np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300)):.3g} times")
