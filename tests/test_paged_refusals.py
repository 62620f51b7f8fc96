"""What the paged operators refuse, checked without a device: every argument is looked at before the device is touched, so a call
with a NULL device and made-up pointers ends with the argument's own message, and a call that is right with the device's."""
import ctypes as C

import pytest

from kalosm_amd import _lib
from kalosm_amd.fusor import FusorHipError, PagedBatch, PagedKvCache, RopeCache, Tensor

INVALID, UNSUPPORTED = _lib.FH_ERR_INVALID, _lib.FH_ERR_UNSUPPORTED
P = 4096  # a pointer that is aligned and never followed

ATTENTION = dict(dtype=1, kv_dtype=1, q=P, q_st=512, q_sh=64, hq=8, hkv=2, d=64, scale=0.125, window=0, k=P, v=P, page=2048, head=1024, slot=64,
                 pages=9, page_size=16, starts=P, lens=P, table=P, cols=4, seqs=2, tokens=5, max_new=3, max_len=0, out=2 * P)
APPEND = dict(dtype=1, kv_dtype=1, q=P, q_st=512, q_sh=64, kr=P, vr=P, kv_st=128, kv_sh=64, hq=8, hkv=2, d=64, cos=P, sin=P, rows=64, pairs=32, positions=None,
              sections=None, axes=1, interleaved=0, k=P, v=P, page=2048, head=1024, slot=64, pages=9, page_size=16, starts=P, lens=P, table=P,
              cols=4, seqs=2, tokens=5, out=P)

SHARED = [
    (dict(k=0), INVALID, "NULL"), (dict(v=0), INVALID, "NULL"), (dict(lens=0), INVALID, "NULL"), (dict(table=0), INVALID, "NULL"),
    (dict(dtype=7), INVALID, "not type 7"), (dict(kv_dtype=-1), INVALID, "not type -1"), (dict(dtype=2), UNSUPPORTED, "the same type"),
    (dict(dtype=1, kv_dtype=0), UNSUPPORTED, "the same type"), (dict(hq=7), INVALID, "evenly"), (dict(hkv=0), INVALID, "evenly"),
    (dict(d=68), UNSUPPORTED, "head_dim 68"), (dict(d=264, page=1 << 16, head=1 << 13, slot=264), UNSUPPORTED, "head_dim 264"), (dict(d=-8), INVALID, "shape"),
    (dict(page_size=8), UNSUPPORTED, "pages of 8"), (dict(page_size=48), UNSUPPORTED, "pages of 48"), (dict(page_size=8192), UNSUPPORTED, "pages of 8192"),
    (dict(pages=0), INVALID, "shape"), (dict(cols=0), INVALID, "shape"), (dict(seqs=-1), INVALID, "shape"), (dict(tokens=-1), INVALID, "shape"),
    (dict(seqs=65536), INVALID, "65535"), (dict(cols=1 << 28), INVALID, "past"), (dict(starts=0), INVALID, "need their starts"),
    (dict(slot=56), INVALID, "strides"), (dict(page=-2048), INVALID, "strides"), (dict(head=512), INVALID, "overlap"), (dict(page=1024), INVALID, "overlap"),
    (dict(k=P + 2), UNSUPPORTED, "16 bytes"), (dict(slot=68, head=1088, page=2176), UNSUPPORTED, "16 bytes"), (dict(page=1 << 60), INVALID, "strides"),
]


def call(name, base, change):
    a = {**base, **change}
    lib = _lib.load()
    status = getattr(lib, name)(None, *[None if v == 0 and isinstance(v, int) and k in ("q", "k", "v", "kr", "vr", "lens", "table", "starts", "out", "cos", "sin") else v
                                        for k, v in a.items()])
    return status, lib.fh_last_error().decode()


@pytest.mark.parametrize("change,status,text", SHARED + [
    (dict(q=0), INVALID, "NULL"), (dict(out=0), INVALID, "NULL"), (dict(scale=0.0), INVALID, "scale"), (dict(scale=float("nan")), INVALID, "scale"),
    (dict(scale=float("inf")), INVALID, "scale"), (dict(window=-1), INVALID, "window"), (dict(max_new=-1), INVALID, "max_new"), (dict(max_len=-1), INVALID, "max_len"),
    (dict(out=P), INVALID, "q cannot be"), (dict(scale=2.0 ** 61), INVALID, "scale"), (dict(scale=2.0 ** -61), INVALID, "scale"), (dict(seqs=65535, cols=1 << 18), INVALID, "2^38"), (dict(hq=65528, seqs=2048, cols=1 << 14), INVALID, "2^38")])
def test_attention(change, status, text):
    got, said = call("fh_paged_attention", ATTENTION, change)
    assert got == status and text in said, (got, said)


@pytest.mark.parametrize("change,status,text", SHARED + [
    (dict(kr=0), INVALID, "NULL"), (dict(vr=0), INVALID, "NULL"), (dict(q=0), INVALID, "together"), (dict(out=0), INVALID, "together"), (dict(cos=0), INVALID, "together"),
    (dict(axes=0), INVALID, "axes"), (dict(axes=5), INVALID, "axes"), (dict(axes=2), INVALID, "several axes"), (dict(rows=0), INVALID, "tables"),
    (dict(pairs=33), INVALID, "sections of 33"), (dict(cos=0, sin=0, positions=P), INVALID, "without tables"),
    (dict(q_st=1024), INVALID, "its own output"), (dict(q_sh=72), INVALID, "its own output"), (dict(tokens=1 << 24), INVALID, "2^24")])
def test_append(change, status, text):
    got, said = call("fh_paged_rope_append", APPEND, change)
    assert got == status and text in said, (got, said)


@pytest.mark.parametrize("sections,text", [((16, -1), "section 1"), ((16, 17), "sections of 33"), ((0, 0), "without a pair")])
def test_sections(sections, text):
    got, said = call("fh_paged_rope_append", APPEND, dict(axes=2, positions=P, sections=(C.c_int32 * 2)(*sections)))
    assert got == INVALID and text in said, (got, said)


def test_what_is_right_wants_its_device():
    for name, base in (("fh_paged_attention", ATTENTION), ("fh_paged_rope_append", APPEND)):
        got, said = call(name, base, {})
        assert got == INVALID and "device" in said, said
        for change in (dict(page=2048, head=64, slot=128), dict(dtype=0), dict(dtype=0, kv_dtype=2), dict(dtype=2, kv_dtype=2), dict(hkv=1, page=1024, head=64)):
            got, said = call(name, base, change)
            assert got == INVALID and "device" in said, (change, said)


def test_tensors_that_do_not_match():
    """Wrong shapes, types and devices on the way in, on devices that are none (nothing here gets as far as a call)."""
    class Nowhere:
        _lib, _h = _lib.load(), None

        def alloc(self, size):
            return P

        def free(self, ptr):
            pass

    here, there = Nowhere(), Nowhere()

    def t(*shape, dtype="f16", device=here):
        return Tensor(device, shape, dtype, ptr=P)

    cache, batch = PagedKvCache.over(t(9, 2, 16, 64), t(9, 2, 16, 64)), PagedBatch(t(3, dtype="i32"), t(3, 4, dtype="i32"))
    q, k = t(3, 8, 64), t(3, 2, 64)
    rope = RopeCache.__new__(RopeCache)
    rope.cos, rope.sin = t(32, 32, dtype="f32"), t(32, 32, dtype="f32")
    for text, call in (("out is", lambda: q.paged_attention(cache, batch, 0.1, out=t(3, 8, 32))), ("out is", lambda: q.paged_attention(cache, batch, 0.1, out=t(3, 8, 64, dtype="f32"))),
                       ("match a batch", lambda: t(4, 8, 64).paged_attention(cache, batch, 0.1)), ("match a batch", lambda: t(3, 8, 32).paged_attention(cache, batch, 0.1)),
                       ("match a batch", lambda: t(3, 8, 64, dtype="i32").paged_attention(cache, batch, 0.1)),
                       ("one device", lambda: t(3, 8, 64, device=there).paged_attention(cache, batch, 0.1)), ("one device", lambda: cache.append(t(3, 2, 64, device=there), k, batch)),
                       ("match a batch", lambda: cache.append(k, t(3, 2, 64, dtype="f32"), batch)), ("match a batch", lambda: cache.append(t(3, 1, 64), t(3, 1, 64), batch)),
                       ("match a batch", lambda: cache.append(t(3, 2, 64, dtype="i32"), t(3, 2, 64, dtype="i32"), batch)),
                       ("does not match k", lambda: rope.forward_paged(t(2, 8, 64), k, k, cache, batch)), ("out is", lambda: rope.forward_paged(q, k, k, cache, batch, out=t(3, 8, 64, dtype="f32"))),
                       ("positions are", lambda: rope.forward_paged(q, k, k, cache, batch, positions=t(1, 2, dtype="i32"))), ("layer 1", lambda: cache.append(k, k, batch, layer=1))):
        with pytest.raises(FusorHipError, match=text):
            call()
    with pytest.raises(FusorHipError, match="lens is i32"):
        PagedBatch(t(2, dtype="i32"), t(3, 4, dtype="i32"))
    with pytest.raises(FusorHipError, match="starts"):
        PagedBatch(t(3, dtype="i32"), t(3, 4, dtype="i32"), t(4, dtype="i32"))
    with pytest.raises(FusorHipError, match="pages of shapes"):
        PagedKvCache.over(t(9, 2, 16, 64), t(9, 2, 16, 32))
