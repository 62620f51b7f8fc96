"""What the paged operators of the Python surface refuse before they call the library: on devices that are none, with made-up pointers."""
import pytest

from kalosm_amd.fusor import FusorHipError, PagedBatch, PagedKvCache, RopeCache, Tensor


class Nowhere:
    """A device whose calls end the test: nothing here gets that far."""
    _h = None

    def alloc(self, size):
        return 4096

    def free(self, ptr):
        pass

    class _lib:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")

    _lib = _lib()


HERE, THERE = Nowhere(), Nowhere()


def t(*shape, dtype="f16", device=HERE):
    return Tensor(device, shape, dtype, ptr=4096)


def i32(*shape, device=HERE):
    return t(*shape, dtype="i32", device=device)


def given(**other):
    """The arguments of a call that is right, on HERE but for those named."""
    at = {name: other.get(name, HERE) for name in ("q", "k", "v", "out", "cache", "batch", "positions", "cos", "sin")}
    d = {name: t(3, 8, 64, device=at[name]) for name in ("q", "out")}
    d.update({name: t(3, 2, 64, device=at[name]) for name in "kv"})
    d["cache"] = PagedKvCache.over(t(9, 2, 16, 64, device=at["cache"]), t(9, 2, 16, 64, device=at["cache"]))
    d["batch"] = PagedBatch(i32(3, device=at["batch"]), i32(3, 4, device=at["batch"]))
    d["positions"] = i32(1, 3, device=at["positions"])
    d["rope"] = RopeCache.__new__(RopeCache)
    d["rope"].device, d["rope"].cos, d["rope"].sin = at["cos"], t(32, 32, dtype="f32", device=at["cos"]), t(32, 32, dtype="f32", device=at["sin"])
    return d


def attention(d):
    d["q"].paged_attention(d["cache"], d["batch"], 0.1, out=d["out"])


def append(d):
    d["cache"].append(d["k"], d["v"], d["batch"])


def turned(d):
    d["rope"].forward_paged(d["q"], d["k"], d["v"], d["cache"], d["batch"], d["positions"], out=d["out"])


@pytest.mark.parametrize("call", [attention, append, turned])
def test_what_is_right_reaches_the_library(call):
    with pytest.raises(AssertionError, match="was called"):
        call(given())


@pytest.mark.parametrize("call,names", [(attention, ("q", "out", "cache", "batch")), (append, ("k", "v", "cache", "batch")),
                                        (turned, ("q", "k", "v", "out", "cache", "batch", "positions", "cos", "sin"))])
def test_tensors_of_another_device(call, names):
    """Another handle is another stream, and may be another GPU: no order between its work and the call's."""
    for name in names:
        with pytest.raises(FusorHipError, match="device"):
            call(given(**{name: THERE}))


def test_a_batch_and_a_cache_are_of_one_device():
    for lens, table, starts in ((THERE, HERE, HERE), (HERE, THERE, HERE), (HERE, HERE, THERE)):
        with pytest.raises(FusorHipError, match="device"):
            PagedBatch(i32(3, device=lens), i32(3, 4, device=table), i32(4, device=starts), tokens=5)
    with pytest.raises(FusorHipError, match="device"):
        PagedKvCache.over(t(9, 2, 16, 64), t(9, 2, 16, 64, device=THERE))


@pytest.mark.parametrize("cos,sin", [(t(32, 32), t(32, 32)), (t(32, 32, dtype="f32"), t(32, 32)), (t(32, 32, dtype="f32"), t(31, 32, dtype="f32")),
                                     (t(32, 32, dtype="f32"), t(32, 16, dtype="f32")), (t(1024, dtype="f32"), t(1024, dtype="f32"))])
def test_tables_that_are_not_read_past_their_end(cos, sin):
    d = given()
    d["rope"].cos, d["rope"].sin = cos, sin  # (put there afterwards)
    with pytest.raises(FusorHipError, match="tables are f32"):
        turned(d)
    if sin.nbytes < cos.nbytes or "f16" in (cos.dtype, sin.dtype):
        with pytest.raises(FusorHipError, match="tables are f32"):
            RopeCache.from_parts(cos, sin)


def test_what_the_calls_were_made_from_stays():
    """A batch and a cache hold pointers and sizes made from their tensors: other tensors or sizes are another batch or cache."""
    d = given()
    for whose, names in (("batch", ("device", "lens", "table", "starts", "tokens", "args")), ("cache", ("device", "k", "v", "dtype", "code", "layers", "pages", "kv_heads", "page_size", "head_dim"))):
        for name in names:
            before = getattr(d[whose], name)
            with pytest.raises(AttributeError):
                setattr(d[whose], name, i32(3))
            assert getattr(d[whose], name) is before
    batch, cache = d["batch"], d["cache"]
    assert (batch.tokens, batch.lens.shape, batch.table.shape, batch.starts) == (3, (3,), (3, 4), None)
    assert (cache.layers, cache.pages, cache.kv_heads, cache.page_size, cache.head_dim, cache.dtype, cache.k.shape) == (1, 9, 2, 16, 64, "f16", (9, 2, 16, 64))
    batch.max_new, batch.max_len = 2, 40  # (these are looked at in every call)
    assert (batch.max_new, batch.max_len) == (2, 40)
