"""Attention over a paged cache where scores are large and negative: what a maximum, and 14 less a maximum, are rounded by must not be in the
weights, on either side of the powers of two, and must not be left behind by a tile whose scores later ones leave far below."""
import numpy as np
import pytest

from pagedgen import Pages, attention_bound, near, pack, unpack
from kalosm_amd.fusor import Tensor

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]
STEPS = [([1] * 24, [100] * 24), ([1] * 3, [2000, 9000, 500]), ([4] * 9, [60] * 9)]
PROMPTS = [([70] * 8, [300] * 8), ([60] * 3, [128] * 3), ([20], [3000])]
LN2 = 0.6931471824645996  # times 1.4426950408889634 this is 1 in f32: scores are whole numbers to base 2


def run(dev, p, scale):
    cache, batch = p.put(dev)
    out = Tensor.filled_bytes(dev, (p.tokens, p.hq, p.d), 0xFF, p.act)
    Tensor.from_slice(dev, p.q, p.act).paged_attention(cache, batch, scale, out=out)
    return unpack(out.as_slice(), p.act)


def whole_scores(dev, act, kept, d, new, lens):
    """q . k = -2^e + offset, whole numbers that f32 holds, as it does every sum on the way and every product with the scale of 1 or a power of two: scores, their
    differences and the weights' exponents are exact, so nothing but the rounding of weights, sums and results is left in the bound (scores of size 0).

    Offsets are multiples of what the scores are rounded by, so that each lies within some 14 of the power or just above: one for each sequence, and from 64 to 64
    positions one more, or 40 more."""
    assert np.float32(LN2) * np.float32(1.4426950408889634) == 1
    p = Pages(d, new, lens, 4, 2, d, 16, act, kept)
    v = unpack(p.v, kept)
    for e in (22, 23, 24, 25, 26, 30):
        ulp = 2.0 ** max(0, e - 24)
        a, b = e // 2, e - e // 2
        for rise in (0, 1, 40):
            if rise * max(lens) // 64 > 2000:
                continue  # (40 a tile would not be exact in f16)
            k, q = np.zeros(p.k.shape), np.zeros(p.q.shape)
            q[:, :, 0], q[:, :, 1], q[:, :, 2] = -2.0 ** a, ulp, ulp
            scores = []
            for i, n in enumerate(lens):
                pos = np.arange(n)
                tile = (pos // 64)[:, None] * np.ones(2)
                at = k[p.table[i, pos // 16], :, pos % 16]
                at[..., 0], at[..., 1], at[..., 2] = 2.0 ** b, i, rise * tile
                k[p.table[i, pos // 16], :, pos % 16] = at
                scores.append(-2.0 ** e + ulp * (i + rise * tile[:, 0]))
            p.k, p.q = pack(k, kept), pack(q, act)
            assert np.array_equal(unpack(p.k, kept), k) and np.array_equal(unpack(p.q, act), q)
            got = run(dev, p, LN2)
            for i, (m, n) in enumerate(zip(new, lens)):
                seen = np.arange(n) <= np.arange(n - m, n)[:, None]
                w = np.where(seen, scores[i], -np.inf)
                w = np.exp2(w - w.max(1, keepdims=True))
                w /= w.sum(1, keepdims=True)
                pos = np.arange(n)
                x = v[p.table[i, pos // 16], :, pos % 16].reshape(n, 2 * d)
                o, mass, whole = (np.repeat((f @ y).reshape(m, 2, d), 2, 1) for f, y in ((w, x), (w, np.abs(x)), (seen, np.abs(x))))
                rows = slice(p.starts[i], p.starts[i + 1])
                near(got[rows], o, attention_bound(o, mass, whole, 0.0, n, d, act, kept), f"2^{e}, {rise} a tile, sequence {i}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", STEPS)
def test_steps_at_whole_scores(dev, act, kept, d, new, lens):
    whole_scores(dev, act, kept, d, new, lens)


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", PROMPTS)
def test_prompts_at_whole_scores(dev, act, kept, d, new, lens):
    whole_scores(dev, act, kept, d, new, lens)


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens,low", [([1] * 24, [100] * 24, 64), ([1] * 2, [9000, 3000], 2048), ([4] * 9, [60] * 9, 48), ([60, 30], [128, 128], 64), ([130, 40], [400, 700], 256),
                                          ([20], [5000], 4096), ([300, 40], [2348, 2100], 2048)])
def test_the_first_positions_far_below(dev, act, kept, d, new, lens, low):
    """The first `low` positions score -2^25 and less (next to f16; else -2^37 and less), the others as usual: weights of the first are 0, and the result is that of
    the others alone, whatever the first tiles' maxima were rounded by."""
    p = Pages(7, new, lens, 8, 2, d, 16, act, kept)
    rng = np.random.default_rng(17)
    k, q = unpack(p.k, kept), unpack(p.q, act)
    far = 3.5e4 if kept == "f16" else 2.0 ** 21
    for i, n in enumerate(lens):
        pos = np.arange(n)
        at = k[p.table[i, pos // 16], :, pos % 16]
        at[..., 0] = np.where(pos < low, -(10000.0 if kept == "f16" else 2.0 ** 20), 0)[:, None]
        k[p.table[i, pos // 16], :, pos % 16] = at
    q[:, :, 0] = far * rng.uniform(0.75, 1.5, q.shape[:2])
    p.k, p.q = pack(k, kept), pack(q, act)
    got = run(dev, p, 0.125)
    p.table[:, :low // 16] = -1  # (of the oracle: positions that are not there)
    want, bound = p.attention(0.125)
    near(got, want, bound, f"{act}/{kept} {d} {new[:2]}")
