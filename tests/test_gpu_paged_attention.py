"""Attention over a paged cache against the definition in 64 bits: one new token a sequence (split over the cache and joined)
and several (tiles of a prompt); slots that nothing may see hold NaN in every case."""
import numpy as np
import pytest

from pagedgen import HALF_STEP, SMALLEST, Pages, near, pack, unpack
from kalosm_amd.fusor import FusorHipError, PagedBatch, PagedKvCache, Tensor

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16")]


def run(dev, p, window=0, q=None, scale=None, **kw):
    cache, batch = p.put(dev)
    for name, value in kw.items():
        setattr(batch, name, value)
    qt = Tensor.from_slice(dev, p.q, p.act) if q is None else q
    out = Tensor.filled_bytes(dev, (p.tokens, p.hq, p.d), 0xFF, p.act)  # NaN where nothing is written
    qt.paged_attention(cache, batch, scale or p.d ** -0.5, window=window, out=out)
    return unpack(out.as_slice(), p.act)


def check(dev, p, window=0, what="", scale=None, **kw):
    got = run(dev, p, window, scale=scale, **kw)
    want, bound = p.attention(scale or p.d ** -0.5, window)
    lo, hi = int(p.starts[0]), int(p.starts[-1])
    near(got[lo:hi], want[lo:hi], bound[lo:hi], what)
    assert np.isnan(got[:lo]).all() and np.isnan(got[hi:]).all(), f"{what}: rows of no sequence were written"


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (5, 1, 64), (4, 4, 96), (16, 1, 128), (3, 3, 8), (40, 2, 256), (6, 2, 200), (18, 1, 72)])
def test_step_heads(dev, act, kept, hq, hkv, d):
    lens = [1, 2, 15, 16, 17, 31, 33, 300]
    check(dev, Pages(hq + d, [1] * len(lens), lens, hq, hkv, d, 16, act, kept), what=f"{act}/{kept} {hq}/{hkv} of {d}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 256, 4096])
def test_step_pages(dev, act, kept, page):
    lens = [page - 1, page, page + 1, 2 * page + 5, 1]
    check(dev, Pages(page, [1] * len(lens), lens, 8, 2, 64, page, act, kept), what=f"{act}/{kept} pages of {page}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("lens", [[4097], [20011], [5000, 1, 0, 700, 2048, 64, 9, 6001]])
def test_step_long(dev, act, kept, lens):
    check(dev, Pages(len(lens), [1] * len(lens), lens, 8, 2, 128, 64, act, kept), what=f"{act}/{kept} {lens}")


def test_step_many_sequences(dev):
    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 90, 333)]
    check(dev, Pages(9, [1] * len(lens), lens, 4, 2, 64, 16, "f16", "f16"), what="333 short sequences")
    check(dev, Pages(9, [1] * len(lens), lens, 4, 4, 128, 32, "bf16", "bf16"), what="333 short sequences, a head each")


@pytest.mark.parametrize("new", [[1, 1, 1], [7, 1, 33]])
@pytest.mark.parametrize("window", [1, 16, 37, 1000])
@pytest.mark.parametrize("act,kept", [("f16", "f16"), ("f32", "f32"), ("bf16", "bf16")])
def test_window(dev, new, window, act, kept):
    check(dev, Pages(window, new, [777, 1, 130], 8, 2, 64, 16, act, kept), window, what=f"window {window}, rows {new}")


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 130]])
@pytest.mark.parametrize("act,kept", [("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
def test_holes(dev, new, act, kept):
    """Entries that are no page are not seen: below 0, past the pool, in the middle of a sequence, all of one."""
    p = Pages(3, new, [700, 65, 130], 8, 2, 128, 16, act, kept)
    p.table[0, 3], p.table[0, 17], p.table[0, 30:33] = -1, p.pages, (2 ** 31 - 1, -2 ** 31, p.pages + 7)
    p.table[1, :] = -5
    p.table[2, 0] = -1
    check(dev, p, what=f"holes, rows {new}")
    check(dev, p, 64, what=f"holes and a window, rows {new}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (5, 1, 64), (4, 4, 96), (7, 1, 128), (3, 3, 8), (2, 1, 256), (6, 2, 200)])
def test_prompt_heads(dev, act, kept, hq, hkv, d):
    p = Pages(hq + d, [70, 2, 129, 1, 31], [70, 90, 140, 1, 300], hq, hkv, d, 16, act, kept)
    check(dev, p, what=f"{act}/{kept} {hq}/{hkv} of {d}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("new,lens", [([2], [2]), ([64], [64]), ([65], [65]), ([128], [129]), ([300], [300]), ([5], [3000]), ([257, 255], [257, 1200])])
def test_prompt_lengths(dev, act, kept, new, lens):
    check(dev, Pages(sum(lens), new, lens, 4, 1, 128, 32, act, kept), what=f"{act}/{kept} {new} of {lens}")


@pytest.mark.parametrize("page", [16, 32, 64, 256, 4096])
@pytest.mark.parametrize("act,kept", [("f16", "f16"), ("f32", "f32")])
def test_prompt_pages(dev, page, act, kept):
    check(dev, Pages(page, [100, 3], [page + 37, 2 * page - 1], 4, 2, 64, page, act, kept), what=f"pages of {page}")


@pytest.mark.parametrize("new", [[1, 1, 1], [5, 0, 40]])
@pytest.mark.parametrize("act,kept", [("f16", "f16"), ("f32", "f32"), ("f32", "f16"), ("bf16", "bf16")])
def test_slot_major_pages_and_rows_of_no_sequence(dev, new, act, kept):
    p = Pages(11, new, [200, 17, 90], 6, 3, 64, 16, act, kept, slot_major=True, before=3, behind=4)
    check(dev, p, what="pages [page][slot][head]")


@pytest.mark.parametrize("new", [[1, 1], [20, 130]])
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
def test_rows_of_a_fused_projection(dev, new, act):
    """q is a view: other strides, and an odd beginning."""
    p = Pages(12, new, [150, 333], 4, 2, 128, 16, act, act)
    wide = np.zeros((p.tokens, 8 * 128 + 1), p.q.dtype)
    wide[:, 1:513] = p.q.reshape(p.tokens, 512)
    t = Tensor.from_slice(dev, wide.reshape(-1), act)
    view = Tensor(dev, p.q.shape, act, ptr=t.ptr + wide.itemsize)
    cache, batch = p.put(dev)
    out = view.paged_attention(cache, batch, 128 ** -0.5, strides=(8 * 128 + 1, 128))
    want, bound = p.attention(128 ** -0.5)
    near(unpack(out.as_slice(), act), want, bound, f"a view of {act}")


@pytest.mark.parametrize("new", [[1, 1], [50, 3]])
@pytest.mark.parametrize("act,kept", TYPES)
def test_sharp_and_large_values(dev, new, act, kept):
    """Scores far apart, and values next to the ends of the types' ranges."""
    p = Pages(21, new, [900, 70], 4, 2, 64, 16, act, kept, spread=30.0)
    check(dev, p, what="scores of some hundreds")
    p.v = np.where(np.isnan(unpack(p.v, kept)), p.v, {"f16": lambda a: (a * np.float16(2 ** -14)), "f32": lambda a: a * np.float32(1e30), "bf16": lambda a: a}[kept](p.v)).astype(p.v.dtype)
    check(dev, p, what="values of another size")


@pytest.mark.parametrize("act,kept", TYPES)
def test_infinite_and_nan_rows_stay_theirs(dev, act, kept):
    """An infinity or a NaN in V reaches the rows that see it, and no others."""
    for new in ([1, 1, 1], [90, 1, 70]):
        p = Pages(31, new, [90, 200, 300], 4, 2, 64, 16, act, kept)
        inf = {"f32": np.float32(np.inf), "f16": np.float16(np.inf), "bf16": np.uint16(0x7F80)}[kept]
        nan = {"f32": np.float32(np.nan), "f16": np.float16(np.nan), "bf16": np.uint16(0x7FC0)}[kept]

        def at(a, i, pos):
            return a[p.table[i, pos // 16], :, pos % 16]

        at(p.v, 0, 89)[:, 5] = nan   # only the last row of the first sequence sees it
        at(p.v, 2, 290)[:, 7] = inf
        got = run(dev, p)
        with np.errstate(invalid="ignore"):
            want, bound = p.attention(64 ** -0.5)
        fine = np.isfinite(want)
        assert (np.isfinite(got) == fine).all(), f"{new}: {np.argwhere(np.isfinite(got) != fine)[:5].tolist()}"
        near(np.where(fine, got, 0), np.where(fine, want, 0), np.where(fine, bound, 1), f"{act}/{kept} {new}")


@pytest.mark.parametrize("new", [[1] * 5, [40, 3, 1, 0, 65]])
def test_max_len_only_chooses(dev, new):
    p = Pages(41, new, [900, 3, 4100, 64, 65], 8, 2, 128, 32, "f16", "f16")
    want, bound = p.attention(128 ** -0.5)
    for n in (0, 1, 100, 4100, 1 << 20):
        got = run(dev, p, max_len=n)
        near(got, want, bound, f"max_len {n}")


def test_one_row_each_without_starts(dev):
    p = Pages(51, [1, 1, 1], [10, 500, 77], 4, 2, 64, 16, "f16", "f16")
    cache, batch = p.put(dev)
    alone = PagedBatch(batch.lens, batch.table)
    q = Tensor.from_slice(dev, p.q, "f16")
    a, b = (q.paged_attention(cache, x, 0.125).as_slice() for x in (batch, alone))
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))


def test_lengths_that_do_not_fit_are_safe(dev):
    """Lengths past the table, below the new rows and below 0; starts past the rows."""
    p = Pages(61, [1, 4, 2], [40, 60, 30], 4, 2, 64, 16, "f16", "f16")
    cache, batch = p.put(dev)
    q = Tensor.from_slice(dev, p.q, "f16")
    want, bound = p.attention(0.125)
    for lens in ([2 ** 31 - 1, 60, -7], [10 ** 6, 2, 0]):
        b = PagedBatch(Tensor.from_slice(dev, np.array(lens, np.int32), "i32"), batch.table, batch.starts, tokens=p.tokens, max_new=4)
        got = unpack(q.paged_attention(cache, b, 0.125).as_slice(), "f16")
        if lens[1] == 60:
            near(got[1:5], want[1:5], bound[1:5], "the others")
        else:
            assert (got[1:3] == 0).all()  # positions below 0 see nothing
        assert (got[5:] == 0).all()
    starts = Tensor.from_slice(dev, np.array([-4, 1, 5, 100], np.int32), "i32")
    b = PagedBatch(batch.lens, batch.table, starts, tokens=p.tokens, max_new=50)
    near(unpack(q.paged_attention(cache, b, 0.125).as_slice(), "f16")[1:5], want[1:5], bound[1:5], "rows of the middle sequence")


def test_graphs_share_their_scratch(dev):
    """Two captured calls and an eager one in between, replayed in turn with lengths that change."""
    a = Pages(71, [1, 1], [3000, 400], 8, 2, 128, 32, "f16", "f16")
    b = Pages(72, [50], [5000], 8, 2, 128, 32, "bf16", "bf16")
    made = []
    for p in (a, b):
        cache, batch = p.put(dev)
        q, out = Tensor.from_slice(dev, p.q, p.act), Tensor.zeros(dev, p.q.shape, p.act)
        q.paged_attention(cache, batch, 128 ** -0.5, out=out)
        made.append((p, cache, batch, q, out))
    graphs = []
    for p, cache, batch, q, out in made:
        dev.graph_begin()
        q.paged_attention(cache, batch, 128 ** -0.5, out=out)
        graphs.append(dev.graph_end())
    for turn in range(3):
        for (p, cache, batch, q, out), graph in zip(made, graphs):
            p.lens = [x - 37 * turn for x in p.lens]
            t = np.array(p.lens, np.int32)
            from kalosm_amd import _lib
            _lib.check(dev._lib.fh_upload(dev._h, batch.lens.ptr, t.ctypes.data, t.nbytes))
            graph.launch()
            want, bound = p.attention(128 ** -0.5)
            near(unpack(out.as_slice(), p.act), want, bound, f"replay {turn}")
            q.paged_attention(cache, batch, 128 ** -0.5, out=out)
            near(unpack(out.as_slice(), p.act), want, bound, f"eager {turn}")
            p.lens = [x + 37 * turn for x in p.lens]


def test_same_call_same_bits(dev):
    for new in ([1] * 9, [33] * 9):
        p = Pages(81, new, [100 * i + 40 for i in range(9)], 8, 2, 128, 16, "f32", "f16")
        first = run(dev, p)
        for _ in range(3):
            assert np.array_equal(run(dev, p), first)


def test_refused(dev):
    p = Pages(91, [1], [20], 4, 2, 64, 16, "f16", "f16")
    cache, batch = p.put(dev)
    with pytest.raises(FusorHipError, match="match a batch"):
        Tensor.zeros(dev, (2, 4, 64), "f16").paged_attention(cache, batch, 0.1)
    with pytest.raises(FusorHipError, match="rows of type"):
        Tensor.zeros(dev, (1, 4, 64), "bf16").paged_attention(cache, batch, 0.1)
    with pytest.raises(FusorHipError, match="share"):
        Tensor.zeros(dev, (1, 3, 64), "f16").paged_attention(cache, batch, 0.1)
    with pytest.raises(FusorHipError, match="layer 1"):
        Tensor.zeros(dev, (1, 4, 64), "f16").paged_attention(cache, batch, 0.1, layer=1)


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("hq,hkv,new", [(8, 2, [4, 1, 3, 0, 4]), (2, 2, [16, 2, 7, 16, 1]), (5, 1, [3, 3, 1, 2, 3]), (8, 1, [2, 2, 0, 1, 2])])
@pytest.mark.parametrize("d", [64, 128, 200])
def test_few_rows(dev, act, kept, hq, hkv, new, d):
    """Up to 16 rows of a KV head's heads behind short caches: columns of one tile, each with a limit of its own."""
    lens = [90, 1, 17, 33, 300]
    lens = [max(a, b) for a, b in zip(lens, new)]
    p = Pages(hq + d, new, lens, hq, hkv, d, 16, act, kept)
    check(dev, p, what=f"{new} rows of {hq}/{hkv} heads of {d}")
    check(dev, p, 9, what=f"{new} rows of {hq}/{hkv} heads of {d}, a window of 9")
    p.table[0, 2], p.table[4, 0], p.table[4, 7] = -1, p.pages, -3
    check(dev, p, what=f"{new} rows, holes")


@pytest.mark.parametrize("act,kept", TYPES)
def test_infinities_and_nan_of_few_rows(dev, act, kept):
    """A row does not see what its neighbour behind it sees, whatever that is."""
    for new in ([3, 1, 2], [4, 4, 4]):
        p = Pages(33, new, [90, 40, 300], 4, 2, 64, 16, act, kept)
        for i, bits in ((0, np.nan), (2, np.inf), (1, -np.inf)):
            pos = p.lens[i] - 1
            p.v[p.table[i, pos // 16], :, pos % 16, 5 + i] = pack(np.full(2, bits), kept)
        got = run(dev, p)
        with np.errstate(invalid="ignore"):
            want, bound = p.attention(64 ** -0.5)
        fine = np.isfinite(want)
        assert (~fine).sum() == 3 * 4 and (np.isfinite(got) == fine).all(), f"{new}: {np.argwhere(np.isfinite(got) != fine)[:5].tolist()}"
        near(np.where(fine, got, 0), np.where(fine, want, 0), np.where(fine, bound, 1), f"{act}/{kept} {new}")


@pytest.mark.parametrize("act,kept", [("f16", "f16"), ("f32", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (18, 1)])
def test_a_hundred_ragged_sequences(dev, act, kept, hq, hkv):
    """More sequences than a wavefront has lanes, long and empty ones among them: the line's stretches begin anywhere."""
    rng = np.random.default_rng(7)
    lens = [int(x) for x in rng.integers(0, 200, 150)]
    lens[3], lens[70], lens[71], lens[140] = 3000, 2500, 0, 4111
    new = [1] * 150
    new[5], new[64], new[149] = 0, 0, 0
    p = Pages(14, new, lens, hq, hkv, 64, 32, act, kept)
    check(dev, p, what="150 sequences")
    check(dev, p, 2100, what="150 sequences, a window")
    p.table[3, 20:40], p.table[140, 0], p.table[140, 128] = -1, -1, -1
    check(dev, p, what="150 sequences, holes")


def test_more_sequences_than_sorted(dev):
    """Prompts of more workgroups than run at once: the longest first, of up to 64 sequences, and as they come of more."""
    rng = np.random.default_rng(8)
    for n in (40, 64, 65):
        new = [int(x) for x in rng.integers(0, 90, n)]
        lens = [a + int(b) for a, b in zip(new, rng.integers(0, 200, n))]
        lens[1:4] = [lens[0]] * 3  # equals
        new[1:4] = [min(x, lens[0]) for x in new[1:4]]
        p = Pages(n, new, lens, 16, 8, 64, 16, "bf16", "bf16")
        check(dev, p, what=f"{n} prompts")


def test_a_pool_of_more_than_four_gigabytes(dev):
    """Pages whose bytes lie past 2^32, written and read."""
    pages, page, d = 2200, 1024, 128
    pool = Tensor(dev, (pages, 8, page, d), "f16")  # 4.6 GB, K and V alike
    from kalosm_amd.fusor import PagedKvCache
    cache = PagedKvCache.over(pool, pool)
    rng = np.random.default_rng(9)
    for new in ([1, 1], [40, 1100]):
        table = np.array([[2199, 0], [2150, 2197]], np.int32)
        n = sum(new)
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        batch = PagedBatch(Tensor.from_slice(dev, np.array(new, np.int32), "i32"), Tensor.from_slice(dev, table, "i32"), Tensor.from_slice(dev, starts, "i32"),
                           tokens=n, max_new=max(new), max_len=max(new))
        k = pack(rng.standard_normal((n, 8, d)), "f16")
        q = pack(rng.standard_normal((n, 8, d)), "f16")
        kt = Tensor.from_slice(dev, k, "f16")
        cache.append(kt, kt, batch)
        got = unpack(Tensor.from_slice(dev, q, "f16").paged_attention(cache, batch, d ** -0.5).as_slice(), "f16")
        for i, m in enumerate(new):
            x, y = unpack(q[starts[i]:starts[i + 1]], "f16"), unpack(k[starts[i]:starts[i + 1]], "f16")
            s = np.einsum("ahd,bhd->hab", x, y) * d ** -0.5
            s[:, np.triu(np.ones((m, m), bool), 1)] = -np.inf
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            want = np.einsum("hab,bhd->ahd", w, y)
            # weights and results rounded to f16: half a step each of at most sum w |v|
            assert np.abs(got[starts[i]:starts[i + 1]] - want).max() <= 2.1 * 2.0 ** -11 * np.abs(y).max(), (new, i)


def test_without_scratch_memory(dev):
    """Prompts that cannot have memory for their parts run in one; a captured call as well."""
    p = Pages(17, [20], [3000], 4, 1, 128, 16, "bf16", "bf16")
    from kalosm_amd.fusor import Device
    alone = Device.gpu(0)
    alone.set_option("scratch_limit", 1)
    cache, batch = p.put(alone)
    q, out = Tensor.from_slice(alone, p.q, p.act), Tensor.zeros(alone, p.q.shape, p.act)
    want, bound = p.attention(128 ** -0.5)
    q.paged_attention(cache, batch, 128 ** -0.5, out=out)
    near(unpack(out.as_slice(), p.act), want, bound, "no scratch memory")
    alone.graph_begin()
    q.paged_attention(cache, batch, 128 ** -0.5, out=out)
    g = alone.graph_end()
    for _ in range(3):
        g.launch()
        near(unpack(out.as_slice(), p.act), want, bound, "no scratch memory, captured")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("new,lens", [([100, 40], [400, 40]), ([4, 2], [400, 9]), ([70], [3000])])
@pytest.mark.parametrize("window", [0, 80])
def test_nan_rows_anywhere(dev, act, kept, new, lens, window):
    """Positions that hold nothing but NaN: in front of every row, between the rows, behind a window's beginning, everywhere."""
    p = Pages(35, new, lens, 4, 2, 64, 16, act, kept)
    nan = pack(np.array(np.nan), kept)

    def spoil(i, pos):
        for a in (p.k, p.v):
            a[p.table[i, pos // 16], :, pos % 16] = nan

    for places in ([(0, lens[0] - 2)], [(0, lens[0] - 30)], [(0, lens[0] - 90)], [(0, 5)], [(i, q) for i in range(len(lens)) for q in range(lens[i])]):
        for i, pos in places:
            spoil(i, pos)
        got = run(dev, p, window)
        want, bound = p.attention(64 ** -0.5, window)
        fine = np.isfinite(want)
        assert (np.isfinite(got) == fine).all(), f"{places[:1]}: {np.argwhere(np.isfinite(got) != fine)[:5].tolist()}"
        near(np.where(fine, got, 0), np.where(fine, want, 0), np.where(fine, bound, 1), f"{act}/{kept} {new} {places[:1]}")


@pytest.mark.parametrize("act", ["f16", "f32"])
@pytest.mark.parametrize("d", [64, 200])
@pytest.mark.parametrize("new,lens", [([1] * 24, [100] * 24), ([1, 1], [9000, 3000]), ([4] * 9, [60] * 9), ([300, 100], [300, 900])])
def test_scores_past_the_steps_of_their_sums(dev, act, d, new, lens):
    """Scores of 2^23 to 2^29, where the largest, and 14 - the largest, are rounded by up to 32: the one that is largest has all of the weight.

    Its weight in f16, and the result, are each off by half a step at most: together 2 * 2^-11 of the value, and terms of second order and of f32."""
    p = Pages(91, new, lens, 4, 2, d, 16, act, "f16")
    rng = np.random.default_rng(92)
    values = np.arange(0x7100, 0x7C00, dtype=np.uint16).view(np.float16)  # 10240 and more, all different
    p.k[:], p.q[:] = 0, 0
    p.k[:, :, :, 0] = 1
    tops = []
    for i, n in enumerate(lens):
        pos = np.arange(n)
        at = rng.permutation(n)[:len(values)]  # the others stay at 1
        p.k[p.table[i, at // 16], :, at % 16, 0] = rng.permutation(values)[:len(at), None]
        tops.append(np.maximum.accumulate(p.k[p.table[i, pos // 16], 0, pos % 16, 0].astype(np.float64)))
    p.q[:, :, 0] = pack(unpack(pack(rng.uniform(4000, 60000, (p.tokens, 4)), "f16"), "f16"), act)
    got = run(dev, p)
    want = np.zeros_like(got)
    for row, i, last in p.rows():
        j = np.arange(last + 1)
        top = int(j[p.k[p.table[i, j // 16], 0, j % 16, 0].astype(np.float64) == tops[i][last]][0])
        want[row] = np.repeat(unpack(p.v[p.table[i, top // 16], :, top % 16], "f16"), 2, 0)
    near(got, want, 2.01 * 2.0 ** -11 * np.abs(want) + 2.0 ** -24, f"{act} {d} {new[:3]}")


@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", [([150, 40], [150, 700]), ([40], [4000]), ([3, 1], [200, 300])])
@pytest.mark.parametrize("rise", [0.02, 0.11, -0.11, 1.0])
def test_scores_that_rise(dev, act, kept, d, new, lens, rise):
    """Scores that grow a little or much from a tile of positions to the next, and such that fall."""
    p = Pages(93, new, lens, 4, 2, d, 16, act, kept)
    for i, n in enumerate(lens):
        pos = np.arange(n)
        p.k[p.table[i, pos // 16], :, pos % 16, 0] = pack(rise * (pos - n)[:, None] * np.ones(2), kept)
    q = unpack(p.q, act)
    q[:, :, 0] = d ** 0.5 * np.array([1, 0.5, 1, 2])
    p.q = pack(q, act)
    check(dev, p, what=f"{rise} a position")


def test_more_pairs_than_workgroups_of_a_launch(dev):
    """65535 sequences of 260 KV heads, a position each, in pages that they share."""
    seqs, heads, d, pages = 65535, 260, 8, 64
    rng = np.random.default_rng(94)
    v = pack(rng.standard_normal((pages, heads, 16, d)), "f16")
    kt, vt = (Tensor.from_slice(dev, x, "f16") for x in (v[::-1].copy(), v))
    cache = PagedKvCache.over(kt, vt)
    table = (np.arange(seqs) * 7 % pages).astype(np.int32)
    batch = PagedBatch(Tensor.from_slice(dev, np.ones(seqs, np.int32), "i32"), Tensor.from_slice(dev, table[:, None], "i32"), tokens=seqs)
    q = Tensor.from_slice(dev, np.full((seqs, heads, d), 0.5, np.float16), "f16")
    got = q.paged_attention(cache, batch, 0.25).as_slice()
    assert np.array_equal(got.view(np.uint16), v[table, :, 0].view(np.uint16))


@pytest.mark.parametrize("new", [[1, 1], [2, 3], [20, 130]])
@pytest.mark.parametrize("act,kept", TYPES)
@pytest.mark.parametrize("d", [64, 200])
def test_results_at_an_odd_address(dev, new, act, kept, d):
    p = Pages(13, new, [150, 333], 4, 2, d, 16, act, kept)
    cache, batch = p.put(dev)
    n = p.q.size
    room = Tensor.filled_bytes(dev, (n + 8,), 0xFF, act)
    q = Tensor.from_slice(dev, p.q, act)
    q.paged_attention(cache, batch, d ** -0.5, out=Tensor(dev, p.q.shape, act, ptr=room.ptr + 3 * p.q.itemsize))
    want, bound = p.attention(d ** -0.5)
    got = unpack(room.as_slice(), act)
    near(got[3:n + 3].reshape(want.shape), want, bound, f"{act} {d}")
    assert np.isnan(got[:3]).all() and np.isnan(got[n + 3:]).all()


@pytest.mark.parametrize("act,kept", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("d", [64, 128, 200])
@pytest.mark.parametrize("new,lens", [([1] * 24, [100] * 24), ([1, 1], [9000, 3000]), ([4] * 9, [60] * 9), ([300, 100], [300, 900]), ([3], [5000])])
def test_scores_past_the_exponents_of_their_steps(dev, act, kept, d, new, lens):
    """The same up to scores of 2^76, where they are rounded by 2^52: a weight's exponent must not have that in it."""
    p = Pages(95, new, lens, 4, 2, d, 16, act, kept)
    rng = np.random.default_rng(96)
    values = (np.arange(0x4F00, 0x5F00, dtype=np.uint32) << 16).view(np.float32)  # 2^31 to 2^63, each 1 / 256 or more above the one before
    k = np.zeros(p.k.shape)
    k[:, :, :, 0] = 1
    for i, n in enumerate(lens):
        at = rng.permutation(n)[:2000]
        k[p.table[i, at // 16], :, at % 16, 0] = rng.permutation(values)[:len(at), None]
    p.k = pack(k, kept)
    q = np.zeros(p.q.shape)
    q[:, :, 0] = rng.uniform(4000, 60000, (p.tokens, 4))
    p.q = pack(q, act)
    got = run(dev, p)
    want = np.zeros_like(got)
    for row, i, last in p.rows():
        j = np.arange(last + 1)
        top = int(np.argmax(k[p.table[i, j // 16], 0, j % 16, 0]))
        want[row] = np.repeat(unpack(p.v[p.table[i, top // 16], :, top % 16], kept), 2, 0)
    weight = HALF_STEP[kept] if act == kept else 2.0 ** -22
    near(got, want, 1.01 * (HALF_STEP[act] + weight + 2.0 ** -22) * np.abs(want) + SMALLEST[act], f"{act} {kept} {d} {new[:3]}")
