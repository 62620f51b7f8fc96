"""The paged operators together, as a server uses them: prompts of several sequences in parts, then steps of single tokens with pages handed out as they
are needed and given back behind a window, against the same attention over dense rows in 64 bits; and beside the dense cache's operators."""
import numpy as np
import pytest

from pagedgen import HALF_STEP, pack, unpack
from kalosm_amd.fusor import KvCache, MaskKind, PagedBatch, PagedKvCache, RopeCache, Tensor

pytestmark = pytest.mark.gpu


class Server:
    """Rows of random projections for `n` sequences, and what the pages hold of them."""

    def __init__(self, dev, n, hq, hkv, d, page, dtype, window=0):
        self.dev, self.n, self.hq, self.hkv, self.d, self.page, self.dtype, self.window = dev, n, hq, hkv, d, page, dtype, window
        self.cols, self.rng = 24, np.random.default_rng(3)
        self.pool = list(range(n * self.cols))
        self.rng.shuffle(self.pool)
        self.cache = PagedKvCache(dev, 2, hkv, d, len(self.pool), page, dtype)
        self.table = np.full((n, self.cols), -1, np.int32)
        self.lens = [0] * n
        self.rope = RopeCache.new(d, self.cols * page, 10000.0, dev)
        self.cos, self.sin = self.rope.cos.as_slice().astype(np.float64), self.rope.sin.as_slice().astype(np.float64)
        self.k = [np.zeros((0, hkv, d)) for _ in range(n)]
        self.v = [np.zeros((0, hkv, d)) for _ in range(n)]

    def turn(self, x, pos):
        c, s = self.cos[pos][:, None], self.sin[pos][:, None]
        y = x.copy()
        y[..., 0::2], y[..., 1::2] = x[..., 0::2] * c - x[..., 1::2] * s, x[..., 0::2] * s + x[..., 1::2] * c
        return y

    def step(self, new):
        """New rows of every sequence through both layers of the cache; returns the results and what they should be."""
        for i, m in enumerate(new):
            for c in range(-(-(self.lens[i] + m) // self.page)):
                if self.table[i, c] < 0 and (c + 1) * self.page > self.lens[i]:
                    self.table[i, c] = self.pool.pop()
            self.lens[i] += m
        rows = pack(self.rng.standard_normal((sum(new), self.hq + 2 * self.hkv, self.d)), self.dtype)
        wide = (self.hq + 2 * self.hkv) * self.d
        t = Tensor.from_slice(self.dev, rows.reshape(-1), self.dtype)
        q, k, v = (Tensor(self.dev, (sum(new), h, self.d), self.dtype, ptr=t.ptr + at * self.d * rows.itemsize) for h, at in
                   ((self.hq, 0), (self.hkv, self.hq), (self.hkv, self.hq + self.hkv)))
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        batch = PagedBatch(Tensor.from_slice(self.dev, np.array(self.lens, np.int32), "i32"), Tensor.from_slice(self.dev, self.table, "i32"),
                           Tensor.from_slice(self.dev, starts, "i32"), tokens=sum(new), max_new=max(new), max_len=max(self.lens))
        outs = []
        for layer in range(2):
            turned = self.rope.forward_paged(q, k, v, self.cache, batch, interleaved=True, layer=layer, strides=(wide, self.d))
            outs.append(unpack(turned.paged_attention(self.cache, batch, self.d ** -0.5, self.window, layer).as_slice(), self.dtype))
        x, wants = unpack(rows, self.dtype), []
        for i, m in enumerate(new):
            mine = x[starts[i]:starts[i + 1]]
            pos = np.arange(self.lens[i] - m, self.lens[i])
            self.k[i] = np.concatenate([self.k[i], self.turn(mine[:, self.hq:self.hq + self.hkv], pos)])
            self.v[i] = np.concatenate([self.v[i], mine[:, self.hq + self.hkv:]])
            g = self.hq // self.hkv
            want = np.zeros((m, self.hq, self.d))
            for r, (row, p) in enumerate(zip(self.turn(mine[:, :self.hq], pos), pos)):
                lo = max(0, p - self.window + 1) if self.window else 0
                for h in range(self.hq):
                    s = self.k[i][lo:p + 1, h // g] @ row[h] * self.d ** -0.5
                    w = np.exp(s - s.max())
                    want[r, h] = w @ self.v[i][lo:p + 1, h // g] / w.sum()
            wants.append(want)
        if self.window:  # pages that no row will see again
            for i in range(self.n):
                for c in range(max(0, self.lens[i] - self.window) // self.page):
                    if self.table[i, c] >= 0:
                        self.pool.append(int(self.table[i, c]))
                        self.table[i, c] = -1
        return outs, np.concatenate(wants)


@pytest.mark.parametrize("dtype,window", [("f32", 0), ("f16", 0), ("bf16", 0), ("f16", 40), ("f32", 40)])
def test_prompts_in_parts_then_single_tokens(dev, dtype, window):
    """Q and K are rounded to the type behind their rotation (half a step each of |q|, |k|: 2 half steps of sum |q k| of a score, which is at most
    some 4 sqrt(d) sqrt(d) here, scaled by d^-0.5), weights and results by half a step; scores off by ds change weights by a factor within e^(2 ds)."""
    s = Server(dev, 3, 8, 2, 64, 16, dtype, window)
    for new in ([70, 1, 33], [50, 64, 2], [1, 1, 1], [1, 0, 1], [1, 1, 1], [3, 2, 4], [1, 1, 1], [40, 1, 1], [1, 1, 1]):
        outs, want = s.step(new)
        half = HALF_STEP[dtype]
        ds = 2 * half * 4 * 64 * 64 ** -0.5
        allowed = 1.01 * (np.expm1(2 * ds) + 3 * half + 2.0 ** -18) * 4.5  # (values within 4.5)
        for layer, got in enumerate(outs):
            assert np.abs(got - want).max() <= allowed, f"{dtype} {new} layer {layer}: off by {np.abs(got - want).max():.3g}, allowed {allowed:.3g}"
    if window:
        assert (s.table[:2, 0] == -1).all(), "pages behind the window were given back"  # (the third sequence ends at 45: 45 - 40 < 16)


def test_beside_the_dense_cache(dev):
    """The same sequence through KvCache and flash_attention, and through pages: f32 within its rounding."""
    n, hq, hkv, d = 200, 8, 2, 128
    rng = np.random.default_rng(5)
    q, k, v = (rng.standard_normal((n, h, d)).astype(np.float32) for h in (hq, hkv, hkv))
    dense = KvCache(dev, 1, hkv, d, 512)
    dense.append(0, *(Tensor.from_slice(dev, np.ascontiguousarray(x.transpose(1, 0, 2))) for x in (k, v)))
    ln, cap, kt, vt = dense.view(0)
    keys, values = (Tensor.from_slice(dev, x.as_slice()[None, :, :n]) for x in (kt, vt))
    want = Tensor.from_slice(dev, q.transpose(1, 0, 2)[None]).flash_attention(keys, values, d ** -0.5, mask=MaskKind.Causal).as_slice()[0].transpose(1, 0, 2)
    cache = PagedKvCache(dev, 1, hkv, d, 20, 32, "f32")
    batch = PagedBatch(Tensor.from_slice(dev, np.array([n]), "i32"), Tensor.from_slice(dev, np.arange(19, 12, -1)[None], "i32"), Tensor.from_slice(dev, np.array([0, n]), "i32"),
                       tokens=n, max_new=n, max_len=n)
    cache.append(Tensor.from_slice(dev, k), Tensor.from_slice(dev, v), batch)
    got = Tensor.from_slice(dev, q).paged_attention(cache, batch, d ** -0.5).as_slice()
    # both keep 2^-21 of a score of at most 60 (sum |q k| d^-0.5 of these rows is below that) and as much of the weights
    assert np.abs(got - want).max() <= 4 * 60 * 2.0 ** -21 * np.abs(v).max()
