"""Calls of the paged operators as programs make them: fewer rows than a sequence has, pools with gaps, and a captured step of all three operators."""
import ctypes as C

import numpy as np
import pytest

from pagedgen import HALF_STEP, SMALLEST, Pages, near, pack, unpack
from kalosm_amd import _lib
from kalosm_amd.fusor import RopeCache, Tensor

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("new,lens,most", [([10, 2, 1, 0], [90, 40, 7, 30], 1), ([10, 2, 1, 0], [5000, 40, 7, 30], 1), ([10, 2, 1, 0], [90, 40, 7, 30], 3),
                                           ([130, 20, 41], [300, 20, 90], 40), ([130, 20], [4000, 20], 17), ([9, 200], [9, 200], 0)])
def test_the_first_rows_of_every_sequence(dev, act, kept, new, lens, most):
    """max_new below what sequences have: its first rows are computed, the others left as they were."""
    p = Pages(sum(lens) + most, new, lens, 8, 2, 64, 16, act, kept, before=2, behind=1)
    cache, batch = p.put(dev)
    batch.max_new = most
    out = Tensor.filled_bytes(dev, p.q.shape, 0xFF, act)
    Tensor.from_slice(dev, p.q, act).paged_attention(cache, batch, 0.125, out=out)
    got = unpack(out.as_slice(), act)
    want, bound = p.attention(0.125)
    mine = np.zeros(p.tokens, bool)
    for i, m in enumerate(new):
        mine[p.starts[i]:p.starts[i] + min(m, most)] = True
    near(got[mine], want[mine], bound[mine], f"{most} of {new}")
    assert np.isnan(got[~mine]).all()


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 1, 40], [130, 2, 3]])
@pytest.mark.parametrize("slot_major", [False, True])
def test_pools_with_gaps(dev, act, kept, new, slot_major):
    """Slots, heads and pages of more elements than they hold, appended to and read through the C entry points; the gaps stay as they were."""
    p = Pages(19, new, [200, 17, 130], 4, 2, 72, 16, act, kept)
    size, slot, wide = p.k.itemsize, 80, 96
    if slot_major:
        head, slot = wide, 2 * wide + 16
        page = 16 * slot + 32
    else:
        head = 16 * slot + 16
        page = 2 * head + 48
    room = np.full((p.pages, page), pack(np.full((), 7.0), kept))

    def views(a):
        return np.lib.stride_tricks.as_strided(a, (p.pages, 2, 16, 72), (page * size, head * size, slot * size, size))

    held = np.zeros((p.pages, page), p.k.dtype)
    views(held)[:] = 1
    inside, pools = held.astype(bool), []
    for a in (p.k, p.v):
        r = room.copy()
        views(r)[:] = a
        pools.append(Tensor.from_slice(dev, r, kept))
    cache, batch = p.put(dev)
    cache._layers = [(pools[0].ptr, pools[1].ptr, page, head, slot, p.pages, 16)]
    rng = np.random.default_rng(20)
    k, v = (pack(rng.standard_normal((p.tokens, 2, 72)), act) for _ in range(2))
    cache.append(Tensor.from_slice(dev, k, act), Tensor.from_slice(dev, v, act), batch)
    for row, i, pos in p.rows():
        p.k[p.table[i, pos // 16], :, pos % 16], p.v[p.table[i, pos // 16], :, pos % 16] = pack(unpack(k[row], act), kept), pack(unpack(v[row], act), kept)
    for pool, want in zip(pools, (p.k, p.v)):
        now = pool.as_slice()
        assert np.array_equal(np.ascontiguousarray(views(now)).view(np.uint8), want.view(np.uint8)), "the slots"
        assert np.array_equal(now[~inside], room[~inside]), "the gaps"
    got = unpack(Tensor.from_slice(dev, p.q, act).paged_attention(cache, batch, 0.1).as_slice(), act)
    want, bound = p.attention(0.1)
    near(got, want, bound, f"{act}/{kept} {new}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [30, 2100, 500]), ([3, 1, 2], [30, 210, 60]), ([40, 1, 7], [90, 900, 7])])
def test_a_captured_step(dev, act, kept, new, lens):
    """Rotation, append and attention captured once and replayed for positions, pages and rows that the program writes in between, eager calls among them."""
    hq, hkv, d = 4, 2, 64
    p = Pages(23, new, [n + 40 for n in lens], hq, hkv, d, 16, act, kept)  # (room for what follows)
    p.lens = list(lens)
    cache, batch = p.put(dev)
    batch.max_len = 0
    rng = np.random.default_rng(24)
    angle = rng.uniform(-3, 3, (max(lens) + 40, d // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    rope = RopeCache.from_parts(Tensor.from_slice(dev, cos), Tensor.from_slice(dev, sin))
    tensors = [Tensor.zeros(dev, (p.tokens, h, d), act) for h in (hq, hkv, hkv, hq, hq)]
    q, k, v, turned, out = tensors

    def step():
        rope.forward_paged(q, k, v, cache, batch, interleaved=True, out=turned)
        turned.paged_attention(cache, batch, d ** -0.5, out=out)

    def upload(t, a):
        a = np.ascontiguousarray(a)
        _lib.check(dev._lib.fh_upload(dev._h, C.c_void_p(t.ptr), a.ctypes.data_as(C.c_void_p), a.nbytes))

    def check(what):
        rows = {name: unpack(t.as_slice(), act) for name, t in (("q", q), ("k", k), ("v", v), ("turned", turned), ("out", out))}
        held = p.held()
        for row, i, pos in p.rows():
            c, s = cos[pos].astype(np.float64), sin[pos].astype(np.float64)
            at = (p.table[i, pos // 16], slice(None), pos % 16)
            for name, got, dtype in (("q", rows["turned"][row], act), ("k", unpack(held[0][at], kept), kept)):
                x = rows[name][row]
                y, inner = np.zeros_like(x), np.zeros_like(x)
                a, b = x[:, 0::2], x[:, 1::2]
                y[:, 0::2], y[:, 1::2] = a * c - b * s, a * s + b * c
                inner[:, 0::2], inner[:, 1::2] = abs(a * c) + abs(b * s), abs(a * s) + abs(b * c)
                inner *= 3 * HALF_STEP["f32"]
                near(got, y, 1.01 * (inner + HALF_STEP[dtype] * (abs(y) + inner)) + SMALLEST[dtype], f"{what}: {name} of row {row}")
            assert np.array_equal(held[1][at], pack(rows["v"][row], kept)), f"{what}: v of row {row}"
        p.k, p.v = held
        p.q = pack(rows["turned"], act)
        want, bound = p.attention(d ** -0.5)
        near(rows["out"], want, bound, what)

    def turn_on(i):
        for t in (q, k, v):
            upload(t, pack(rng.standard_normal(t.shape), act))
        p.lens = [min(a + m, b + 40) for a, m, b in zip(p.lens, new, lens)] if i else p.lens
        order = rng.permutation(p.pages).astype(np.int32)  # the pool moved about: pages and their numbers alike
        kk, vv = (np.empty_like(a) for a in p.held())
        kk[order], vv[order] = p.held()
        upload(p.kt, kk), upload(p.vt, vv)
        p.table = np.where(p.table >= 0, order[np.maximum(p.table, 0)], p.table).astype(np.int32)
        upload(batch.table, p.table), upload(batch.lens, np.array(p.lens, np.int32))

    turn_on(0)
    step()
    check("eager")
    dev.graph_begin()
    step()
    graph = dev.graph_end()
    for i in range(1, 5):
        turn_on(i)
        graph.launch()
        check(f"replay {i}")
        if i == 2:
            turn_on(i)
            step()
            check("eager in between")
