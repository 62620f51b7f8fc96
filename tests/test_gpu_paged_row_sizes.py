"""Rows and scales of any size: f32 rows over f16 pages, which go to the matrix cores brought to 2^14 by a power of two that the scale takes back, and rows as small as
keys are large."""
import numpy as np
import pytest

from pagedgen import Pages, attention_bound, near, pack, unpack
from kalosm_amd.fusor import Tensor

pytestmark = pytest.mark.gpu

BATCHES = [([1] * 24, [100] * 24), ([1] * 2, [9000, 300]), ([4] * 9, [60] * 9), ([70, 20], [300, 90]), ([20], [3000])]


def run(dev, p, scale):
    cache, batch = p.put(dev)
    out = Tensor.filled_bytes(dev, (p.tokens, p.hq, p.d), 0xFF, p.act)
    Tensor.from_slice(dev, p.q, p.act).paged_attention(cache, batch, scale, out=out)
    return unpack(out.as_slice(), p.act)


@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", BATCHES)
@pytest.mark.parametrize("row,scale", [(-76, 60), (-60, 44), (44, -60), (100, -60), (-120, 60)])
def test_small_and_large_rows(dev, d, new, lens, row, scale):
    """q of 2^row and keys such that scores are of some units where keys of f16 can do that; the bound is every row's."""
    p = Pages(5, new, lens, 4, 2, d, 16, "f32", "f16")
    rng = np.random.default_rng(6)
    size = np.clip(-row - scale, -20, 14)
    at = np.isfinite(unpack(p.k, "f16"))
    p.k = np.where(at, pack(2.0 ** size * rng.uniform(-1, 1, p.k.shape), "f16"), p.k)
    p.q = pack(2.0 ** row * rng.standard_normal(p.q.shape), "f32")
    got = run(dev, p, 2.0 ** scale)
    with np.errstate(over="ignore"):
        want, bound = p.attention(2.0 ** scale)
    near(got, want, bound, f"rows of 2^{row}, scale 2^{scale}")


@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", BATCHES)
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_zero_beside_the_largest(dev, d, new, lens, sign):
    """q of 2^90 at a scale of 2^60: keys of 0 have scores of 0, which is no product with infinity, and one of 2^-24 has 2^126: the only one that counts, or (below
    0) the only one that does not.  Scores are exact or without end apart: of size 0 in the bound."""
    p = Pages(8, new, lens, 4, 2, d, 16, "f32", "f16")
    v, k = unpack(p.v, "f16"), np.zeros(p.k.shape)
    first = [(n - m) // 2 for m, n in zip(new, lens)]
    for i, at in enumerate(first):
        k[p.table[i, at // 16], :, at % 16, 3] = sign * 2.0 ** -24
    p.k, p.q = pack(k, "f16"), pack(np.full(p.q.shape, 2.0 ** 90), "f32")
    got = run(dev, p, 2.0 ** 60)
    for row, i, last in p.rows():
        j = np.arange(last + 1)
        if last >= first[i]:
            j = np.array([first[i]]) if sign > 0 else np.delete(j, first[i]) if last else j
        x = v[p.table[i, j // 16], :, j % 16]
        o, mass, whole = (np.repeat(y, 2, 0) for y in (x.mean(0), np.abs(x).mean(0), np.abs(x).sum(0)))
        near(got[row], o, attention_bound(o, mass, whole, 0.0, last + 1, d, "f32", "f16"), f"row {row}")


@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", [([4] * 9, [60] * 9), ([70, 20], [300, 90]), ([20], [3000])])
def test_large_rows_in_front_of_what_they_do_not_see(dev, d, new, lens):
    """q . k of 2^129 to 2^142 at a scale of 2^-60, and V with infinities where the last row alone looks: the others have the values of their largest key, by the tiles
    and where they are worked out again.  Keys are 2^-10 of themselves apart and more, scores 2^56 and more: the largest has all of the weight."""
    p = Pages(9, new, lens, 4, 2, d, 16, "f32", "f16")
    rng = np.random.default_rng(10)
    values = np.arange(0x4400, 0x7B00, dtype=np.uint16).view(np.float16).astype(np.float64)  # 4 to 57344
    v, k = unpack(p.v, "f16"), np.zeros(p.k.shape)
    for i, n in enumerate(lens):
        pos = np.arange(n)
        k[p.table[i, pos // 16], :, pos % 16, 5] = rng.permutation(values)[:n, None]
        v[p.table[i, (n - 1) // 16], :, (n - 1) % 16, 1] = np.inf
    p.k, p.v, p.q = pack(k, "f16"), pack(v, "f16"), pack(np.full(p.q.shape, 2.0 ** 127), "f32")
    got = run(dev, p, 2.0 ** -60)
    for row, i, last in p.rows():
        j = np.arange(last + 1)
        if last + 1 == lens[i]:
            assert not np.isfinite(got[row, :, 1]).any()
            continue
        top = int(np.argmax(k[p.table[i, j // 16], 0, j % 16, 5]))
        o = np.repeat(v[p.table[i, top // 16], :, top % 16], 2, 0)
        near(got[row], o, attention_bound(o, np.abs(o), 0 * o, 0.0, last + 1, d, "f32", "f16"), f"row {row}")


@pytest.mark.parametrize("act,kept", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", [([4] * 9, [60] * 9), ([70, 20], [300, 90]), ([20], [3000])])
def test_small_rows_in_front_of_what_they_do_not_see(dev, act, kept, d, new, lens):
    """q of 2^-124 and keys of 2^124, both of 8 bits: scores of some units, worked out again where only the last row looks at infinities."""
    p = Pages(11, new, lens, 4, 2, d, 16, act, kept)
    rng = np.random.default_rng(12)
    some = [rng.choice([-1, 1], s) * rng.integers(128, 256, s) / 128 for s in (p.q.shape, p.k.shape)]
    k, v = 2.0 ** 124 * some[1], unpack(p.v, kept)
    for i, n in enumerate(lens):
        v[p.table[i, (n - 1) // 16], :, (n - 1) % 16, 1] = np.inf
    p.q, p.k, p.v = pack(2.0 ** -124 * some[0], act), pack(k, kept), pack(v, kept)
    got = run(dev, p, 0.125)
    with np.errstate(invalid="ignore"):
        want, bound = p.attention(0.125)
    fine = np.isfinite(want)
    assert (~fine).sum() == 4 * len(lens) and (np.isfinite(got) == fine).all()
    near(got[fine], want[fine], bound[fine], f"{act}/{kept} {new[:2]}")


@pytest.mark.parametrize("kept", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", BATCHES)
@pytest.mark.parametrize("sign", [1, -1])
def test_rows_of_the_largest_floats(dev, kept, d, new, lens, sign):
    """Rows of f32's largest value, which bf16 would round to infinity: keys of 0 have scores of 0, and one of 2^-100 has 2^28 or -2^28, without end apart from them."""
    p = Pages(13, new, lens, 4, 2, d, 16, "f32", kept)
    v, k = unpack(p.v, kept), np.zeros(p.k.shape)
    first = [(n - m) // 2 for m, n in zip(new, lens)]
    for i, at in enumerate(first):
        k[p.table[i, at // 16], :, at % 16, 3] = sign * 2.0 ** -100
    p.k, p.q = pack(k, kept), np.full(p.q.shape, np.finfo(np.float32).max, np.float32)
    got = run(dev, p, 1.0)
    for row, i, last in p.rows():
        j = np.arange(last + 1)
        if last >= first[i]:
            j = np.array([first[i]]) if sign > 0 else np.delete(j, first[i]) if last else j
        x = v[p.table[i, j // 16], :, j % 16]
        o, mass, whole = (np.repeat(y, 2, 0) for y in (x.mean(0), np.abs(x).mean(0), np.abs(x).sum(0)))
        near(got[row], o, attention_bound(o, mass, whole, 0.0, last + 1, d, "f32", kept), f"row {row}")
