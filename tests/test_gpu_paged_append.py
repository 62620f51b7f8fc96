"""Rotary positions of one or several axes with the append to a paged cache, against the definition in 64 bits."""
import numpy as np
import pytest

from pagedgen import HALF_STEP, SMALLEST, Pages, near, pack, unpack
from kalosm_amd.fusor import FusorHipError, PagedKvCache, RopeCache, Tensor

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


def turn(x, where, cos, sin, sections, interleaved):
    """x [tokens, heads, d] in 64 bits turned by the rows `where` [axes, tokens] of the tables; and the size of the products."""
    n, d = sum(sections), x.shape[-1]
    axis = np.repeat(np.arange(len(sections)), sections)
    c = np.stack([cos[where[a], j] for j, a in enumerate(axis)], 1).astype(np.float64)[:, None]
    s = np.stack([sin[where[a], j] for j, a in enumerate(axis)], 1).astype(np.float64)[:, None]
    i = (np.arange(0, 2 * n, 2), np.arange(1, 2 * n, 2)) if interleaved else (np.arange(n), np.arange(n, 2 * n))
    y, size = x.copy(), np.zeros_like(x)
    a, b = x[..., i[0]], x[..., i[1]]
    y[..., i[0]], y[..., i[1]] = a * c - b * s, a * s + b * c
    size[..., i[0]], size[..., i[1]] = abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)
    return y, size


def bound(y, size, dtype):
    """Two products and a sum, each rounded in f32 (three half steps of what they add), then one rounding to the type."""
    inner = 3 * HALF_STEP["f32"] * size
    return 1.01 * (inner + HALF_STEP[dtype] * (abs(y) + inner)) + SMALLEST[dtype]


def tables(rows, pairs, seed=0):
    a = np.random.default_rng(seed).uniform(-np.pi, np.pi, (rows, pairs))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def check(dev, p, sections=None, positions=None, interleaved=False, pairs=None, wide=0, in_place=False, rows=None, what=""):
    """One append; `wide`: q, k and v are views of one tensor of rows with so many elements more in front."""
    rng = np.random.default_rng(7)
    rows = max(p.lens) if rows is None else rows
    pairs = pairs or (sum(sections) if sections else p.d // 2)
    cos, sin = tables(rows, pairs)
    rope = RopeCache.from_parts(Tensor.from_slice(dev, cos), Tensor.from_slice(dev, sin))
    k, v = (pack(rng.standard_normal((p.tokens, p.hkv, p.d)), p.act) for _ in range(2))
    cache, batch = p.put(dev)
    at = None if positions is None else Tensor.from_slice(dev, positions, "i32")
    before_k, before_v = p.held()
    if wide:
        heads = p.hq + 2 * p.hkv
        w = np.zeros((p.tokens, heads * p.d + wide), p.q.dtype)
        w[:, wide:] = np.concatenate([p.q, k, v], 1).reshape(p.tokens, heads * p.d)
        t = Tensor.from_slice(dev, w.reshape(-1), p.act)
        views = [Tensor(dev, s, p.act, ptr=t.ptr + (wide + o * p.d) * w.itemsize) for s, o in
                 ((p.q.shape, 0), (k.shape, p.hq), (v.shape, p.hq + p.hkv))]
        got = rope.forward_paged(*views, cache, batch, at, sections, interleaved, strides=(w.shape[1], p.d),
                                 out=Tensor.filled_bytes(dev, p.q.shape, 0xFF, p.act))
    else:
        qt = Tensor.from_slice(dev, p.q, p.act)
        out = qt if in_place else Tensor.filled_bytes(dev, p.q.shape, 0xFF, p.act)
        got = rope.forward_paged(qt, Tensor.from_slice(dev, k, p.act), Tensor.from_slice(dev, v, p.act), cache, batch, at, sections, interleaved, out=out)
    got = unpack(got.as_slice(), p.act)
    now_k, now_v = p.held()
    sections = sections or [pairs]
    live = [(r, i, pos) for r, i, pos in p.rows() if pos >= 0 and 0 <= p.table[i, pos // p.page] < p.pages and
            (positions is None and pos < rows or positions is not None and ((positions[:, r] >= 0) & (positions[:, r] < rows)).all())]
    r = np.array([x[0] for x in live], int)
    pos = np.array([x[2] for x in live], int)
    where = np.broadcast_to(pos, (len(sections), len(pos))) if positions is None else positions[:, r]
    y, size = turn(unpack(p.q, p.act)[r], where, cos, sin, sections, interleaved)
    near(got[r], y, bound(y, size, p.act), f"{what} q")
    rest = np.setdiff1d(np.arange(p.tokens), r)
    if in_place:
        assert np.array_equal(got[rest], unpack(p.q, p.act)[rest])
    else:
        assert np.isnan(got[rest]).all(), f"{what}: dropped rows of q were written"
    y, size = turn(unpack(k, p.act)[r], where, cos, sin, sections, interleaved)
    b = bound(y, size, p.kept)
    page = np.array([p.table[i, x // p.page] for _, i, x in live], int)
    near(unpack(now_k, p.kept)[page, :, pos % p.page], y, b, f"{what} k")
    want_v = pack(unpack(v, p.act), p.kept)
    assert np.array_equal(now_v[page, :, pos % p.page], want_v[r]), f"{what} v"
    for now, old in ((now_k, before_k), (now_v, before_v)):  # nothing else moved
        now = now.copy()
        now[page, :, pos % p.page] = old[page, :, pos % p.page]
        assert np.array_equal(np.ascontiguousarray(now).view(np.uint8), np.ascontiguousarray(old).view(np.uint8)), f"{what}: other slots were written"


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (5, 1, 64), (3, 3, 8), (4, 2, 200), (2, 1, 256)])
def test_one_axis(dev, act, kept, interleaved, hq, hkv, d):
    p = Pages(d, [1, 20, 0, 3], [50, 20, 9, 300], hq, hkv, d, 16, act, kept, before=2, behind=3)
    check(dev, p, interleaved=interleaved, what=f"{act}/{kept} {hq}/{hkv} of {d}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,sections", [(128, (16, 24, 24)), (64, (8, 12, 12)), (64, (1, 30, 1)), (128, (16, 0, 5)), (32, (3, 4, 5, 4)), (96, (7,))])
def test_axes(dev, act, kept, interleaved, d, sections):
    """Sections of any size, none among them, and heads that turn in part only."""
    p = Pages(d, [30, 1, 44], [60, 33, 44], 4, 2, d, 32, act, kept)
    pos = np.random.default_rng(3).integers(0, 60, (len(sections), p.tokens)).astype(np.int32)
    check(dev, p, sections, pos, interleaved, what=f"sections {sections}")
    if len(sections) == 1:
        check(dev, p, sections, None, interleaved, pairs=d // 2, what="a part of the tables' columns")


@pytest.mark.parametrize("act,kept", [("f32", "f32"), ("f16", "f16"), ("f32", "bf16")])
def test_rows_that_have_no_place_are_dropped(dev, act, kept):
    p = Pages(4, [5, 40, 1], [5, 40, 17], 4, 2, 64, 16, act, kept)
    p.table[1, 1] = -1
    p.table[2, 1] = p.pages
    check(dev, p, what="holes")
    pos = np.random.default_rng(3).integers(0, 40, (2, p.tokens)).astype(np.int32)
    pos[0, 3], pos[1, 7], pos[0, 9], pos[1, 12] = -1, 40, 2 ** 31 - 1, -2 ** 31
    check(dev, p, (16, 16), pos, what="positions outside the tables")
    check(dev, p, rows=20, what="tables shorter than the sequences")
    q = Pages(4, [5, 40, 3], [5, 40, 17], 4, 2, 64, 16, act, kept)
    q.lens[0] = 2  # shorter than its new rows: the first three have no position
    check(dev, q, rows=64, what="a length below the new rows")


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("wide", [8, 1])
def test_views_of_a_fused_projection(dev, act, wide):
    p = Pages(5, [1, 30], [90, 30], 8, 2, 64, 16, act, act)
    check(dev, p, wide=wide, what=f"rows of {wide} elements more")
    check(dev, p, wide=wide, interleaved=True, what=f"rows of {wide} elements more")


@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_and_slot_major(dev, interleaved):
    check(dev, Pages(6, [1, 30], [90, 30], 8, 2, 64, 16, "f16", "f16", behind=1), in_place=True, interleaved=interleaved, what="in place")
    check(dev, Pages(6, [1, 30], [90, 30], 8, 2, 64, 16, "f32", "f32", slot_major=True), interleaved=interleaved, what="[page][slot][head]")


def test_many_rows(dev):
    check(dev, Pages(8, [700, 1, 300], [800, 1, 4000], 4, 1, 64, 128, "f16", "f16"), what="a thousand rows")
    lens = [int(x) for x in np.random.default_rng(8).integers(1, 60, 200)]
    check(dev, Pages(8, [1] * 200, lens, 4, 1, 64, 16, "bf16", "bf16"), what="two hundred sequences")


@pytest.mark.parametrize("act,kept", TYPES)
def test_append_alone(dev, act, kept):
    p = Pages(9, [3, 20], [50, 20], 2, 2, 64, 16, act, kept)
    k, v = (pack(np.random.default_rng(i).standard_normal((p.tokens, 2, 64)), act) for i in range(2))
    cache, batch = p.put(dev)
    cache.append(Tensor.from_slice(dev, k, act), Tensor.from_slice(dev, v, act), batch)
    for now, new in zip(p.held(), (k, v)):
        for r, i, pos in p.rows():
            assert np.array_equal(now[p.table[i, pos // 16], :, pos % 16], pack(unpack(new[r], act), kept))


def test_layers(dev):
    cache = PagedKvCache(dev, 3, 2, 64, 5, 16, "f16")
    p = Pages(10, [4], [4], 2, 2, 64, 16, "f16", "f16")
    _, batch = p.put(dev)
    k = pack(np.random.default_rng(1).standard_normal((4, 2, 64)), "f16")
    cache.append(Tensor.from_slice(dev, k, "f16"), Tensor.from_slice(dev, k, "f16"), batch, layer=1)
    got = cache.k.as_slice()
    assert (got[[0, 2]] == 0).all() and np.array_equal(got[1, p.table[0, 0], :, :4].transpose(1, 0, 2), k)


def test_refused(dev):
    p = Pages(12, [4], [4], 4, 2, 64, 16, "f16", "f16")
    cache, batch = p.put(dev)
    c = Tensor.zeros(dev, (8, 32))
    rope = RopeCache.from_parts(c, c)
    q, k = Tensor.zeros(dev, (4, 4, 64), "f16"), Tensor.zeros(dev, (4, 2, 64), "f16")
    for kw, text in ((dict(sections=(16, 16)), "several axes need"), (dict(sections=(40,)), "sections of 40 pairs"), (dict(sections=(0,)), "without a pair"),
                     (dict(sections=(33, -1), positions=Tensor.zeros(dev, (2, 4), "i32")), "sections of 33"), (dict(positions=Tensor.zeros(dev, (2, 4), "i32")), "positions are"),
                     (dict(sections=(6,) * 5, positions=Tensor.zeros(dev, (5, 4), "i32")), "5 axes")):
        with pytest.raises(FusorHipError, match=text):
            rope.forward_paged(q, k, k, cache, batch, **kw)
    with pytest.raises(FusorHipError, match="do not match"):
        rope.forward_paged(q, Tensor.zeros(dev, (3, 2, 64), "f16"), k, cache, batch)
