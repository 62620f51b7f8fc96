"""The paged operators together, value by value: what the append left in the pages and in q against the rotation's definition, and the attention against its
definition over just those values, so that the bounds have no rounding of q and k in them and a wrong page, layer or position shows."""
import numpy as np
import pytest

from pagedgen import HALF_STEP, SMALLEST, attention_bound, near, pack, unpack
from kalosm_amd.fusor import PagedBatch, PagedKvCache, RopeCache, Tensor

pytestmark = pytest.mark.gpu

LAYERS, HQ, HKV, D, PAGE, COLS = 2, 8, 2, 64, 16, 24


def turned(x, cos, sin):
    """Pairs (2 j, 2 j + 1) of x [rows, heads, D] turned in 64 bits, and how far the kernel may be off: three half steps of f32, one of the type."""
    c, s = cos[:, None], sin[:, None]
    y, size = np.zeros_like(x), np.zeros_like(x)
    a, b = x[..., 0::2], x[..., 1::2]
    y[..., 0::2], y[..., 1::2] = a * c - b * s, a * s + b * c
    size[..., 0::2], size[..., 1::2] = abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)
    return y, 3 * HALF_STEP["f32"] * size


def rounded(y, inner, dtype):
    return 1.01 * (inner + HALF_STEP[dtype] * (abs(y) + inner)) + SMALLEST[dtype]


def definition(q, k, v, first, window, act, kept):
    """Rows q [m, HQ, D] at positions first .. over k, v [positions, HKV, D]: the result in 64 bits and its bound."""
    g, m, n = HQ // HKV, len(q), len(k)
    p, j = np.arange(first, first + m)[:, None], np.arange(n)
    seen = (j <= p) & ((j > p - window) if window else True)
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(HQ):
        x, y, z = q[:, h], k[:, h // g], v[:, h // g]
        s = np.where(seen, x @ y.T * D ** -0.5, -np.inf)
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        size = np.where(seen, np.abs(x) @ np.abs(y).T * D ** -0.5, 0).max(1, keepdims=True)
        out[:, h] = w @ z
        bound[:, h] = attention_bound(out[:, h], w @ np.abs(z), seen @ np.abs(z), size, n, D, act, kept)
    return out, bound


@pytest.mark.parametrize("act,kept", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("window", [0, 40])
def test_prompts_in_parts_then_single_tokens(dev, act, kept, window):
    rng = np.random.default_rng(3)
    pool = [int(x) for x in rng.permutation(3 * COLS)]
    cache = PagedKvCache(dev, LAYERS, HKV, D, len(pool), PAGE, kept)
    rope = RopeCache.new(D, COLS * PAGE, 10000.0, dev)
    cos, sin = (t.as_slice().astype(np.float64) for t in (rope.cos, rope.sin))
    table, lens = np.full((3, COLS), -1, np.int32), [0, 0, 0]
    kept_k, kept_v = ([[np.zeros((0, HKV, D))] * 3 for _ in range(LAYERS)] for _ in range(2))  # [layer][sequence]: as the pages had it behind its append
    for new in ([70, 1, 33], [50, 64, 2], [1, 1, 1], [1, 0, 1], [1, 1, 1], [3, 2, 4], [1, 1, 1], [40, 1, 1], [1, 1, 1]):
        for i, m in enumerate(new):
            for c in range(lens[i] // PAGE, -(-(lens[i] + m) // PAGE)):
                if table[i, c] < 0:
                    table[i, c] = pool.pop()
            lens[i] += m
        n, starts = sum(new), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        batch = PagedBatch(Tensor.from_slice(dev, np.array(lens), "i32"), Tensor.from_slice(dev, table, "i32"), Tensor.from_slice(dev, starts, "i32"),
                           tokens=n, max_new=max(new), max_len=max(lens))
        seq = np.repeat(np.arange(3), new)
        pos = np.concatenate([np.arange(lens[i] - m, lens[i]) for i, m in enumerate(new)])
        made = []
        for layer in range(LAYERS):  # both before either is looked at; every layer has rows of its own
            rows = pack(rng.standard_normal((n, HQ + 2 * HKV, D)), act)
            t = Tensor.from_slice(dev, rows.reshape(-1), act)
            q, k, v = (Tensor(dev, (n, h, D), act, ptr=t.ptr + at * D * rows.itemsize) for h, at in ((HQ, 0), (HKV, HQ), (HKV, HQ + HKV)))
            q = rope.forward_paged(q, k, v, cache, batch, interleaved=True, layer=layer, strides=((HQ + 2 * HKV) * D, D))
            out = Tensor.filled_bytes(dev, q.shape, 0xFF, act)
            made.append((rows, q, q.paged_attention(cache, batch, D ** -0.5, window, layer, out=out)))
        for layer, (rows, q, out) in enumerate(made):
            x, q, got = unpack(rows, act), unpack(q.as_slice(), act), unpack(out.as_slice(), act)
            y, inner = turned(x[:, :HQ + HKV], cos[pos], sin[pos])
            near(q, y[:, :HQ], rounded(y, inner, act)[:, :HQ], f"{new} layer {layer}: q")
            k, v = (unpack(a.as_slice()[layer][table[seq, pos // PAGE], :, pos % PAGE], kept) for a in (cache.k, cache.v))
            near(k, y[:, HQ:], rounded(y, inner, kept)[:, HQ:], f"{new} layer {layer}: k")
            assert np.array_equal(v, unpack(pack(x[:, HQ + HKV:], kept), kept)), f"{new} layer {layer}: v"
            for i, m in enumerate(new):
                r = slice(starts[i], starts[i + 1])
                kept_k[layer][i], kept_v[layer][i] = np.concatenate([kept_k[layer][i], k[r]]), np.concatenate([kept_v[layer][i], v[r]])
                if not m:
                    continue
                want, bound = definition(q[r], kept_k[layer][i], kept_v[layer][i], lens[i] - m, window, act, kept)
                near(got[r], want, bound, f"{new} layer {layer}, sequence {i}")
                for wrong in (np.zeros_like(want), definition(q[r], kept_k[layer][i], np.roll(kept_v[layer][i], 1, 0), lens[i] - m, window, act, kept)[0]):
                    if lens[i] > 1:
                        assert (np.abs(wrong - want) > bound).mean() > 0.5, f"{new} sequence {i}: the bound lets anything pass"
        if window:  # pages that no row will see again
            for i in range(3):
                for c in range(max(0, lens[i] - window) // PAGE):
                    if table[i, c] >= 0:
                        pool.append(int(table[i, c]))
                        table[i, c] = -1
    if window:
        assert (table[:2, 0] == -1).all(), "pages behind the window were given back"
