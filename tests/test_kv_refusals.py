"""CPU: calls of the token cache that are refused, and those beside them that are not (no HIP call is made)."""
import ctypes as C
import itertools

import pytest
import torch

from test_kv import ARG, call  # noqa: F401  (call: the fixture)


def overlap(rows, heads, rs, hs, d):
    starts = [i * rs + j * hs for i, j in itertools.product(range(rows), range(heads))]
    return any(abs(a - b) < d for a, b in itertools.combinations(starts, 2))


@pytest.mark.parametrize("rows,heads", [(4, 4), (3, 2), (2, 6), (1, 4), (4, 2)])
def test_outputs_overlap_in_no_two_rows(call, rows, heads):  # noqa: F811
    """Both strides together decide it: a row's next head may be the next row's first."""
    call.batch.n_seqs, call.batch.rows = 1, rows
    call.batch.table_width = call.batch.table_stride = 5000
    rc, need = call.size(heads=heads)
    assert rc == 0 and need > 0
    seen = set()
    for rs, hs in itertools.product((128, -128, 129, 200, 255, 256, 300, -384, 512, 640, 1000, 4096), repeat=2):
        call.out.row_stride, call.out.head_stride = rs, hs
        # one that is in order gets as far as the scratch, which is a byte too small
        assert call.attend(heads=heads, size=need - 1) == ARG
        bad = overlap(rows, heads, rs, hs, 128)
        assert ("overlapping" if bad else "scratch") in call.why(), (rs, hs)
        seen.add(bad)
        if rows > 1 and heads == 2:
            call.rows.row_stride, call.rows.head_stride = rs, hs
            if bad:
                rc = call.L.gvdb_kv_read_device(C.byref(call.cache), C.byref(call.batch), C.byref(call.rows), None, None)
                assert rc == ARG and "overlapping" in call.why()
    assert seen == ({False} if rows == 1 else {False, True})


def test_strides_of_any_size(call):  # noqa: F811
    call.batch.table_width = call.batch.table_stride = 5000
    need = call.size()[1]
    for rs, hs, bad in ((-(1 << 63), 1 << 62, True), (1 << 62, -(1 << 63), True), (1 << 62, 1 << 62, True), (-(1 << 63), -(1 << 63), True),
                        ((1 << 63) - 1, -(1 << 63), True), (3 << 60, 1 << 62, False), (-(1 << 63), 1000, False), (128, -(1 << 63), False)):
        call.out.row_stride, call.out.head_stride = rs, hs
        assert call.attend(size=need - 1) == ARG and ("overlapping" if bad else "scratch") in call.why(), (rs, hs)


@pytest.mark.parametrize("top,new,width", [(0, 1, 64), (0, 5, 64), (0, 200, 300), (16, 1, 64), (16, 3, 2000)])
def test_scratch_is_asked_for_each_call(call, top, new, width):  # noqa: F811
    """The answer is what the same call takes, for every batch and length on the way down; a smaller batch may need more."""
    call.cache.kv_heads, call.batch.table_width, call.batch.table_stride = 8, width, width
    call.q.row_stride = call.out.row_stride = 32 * 128
    sizes = {}
    for seqs, max_len, cu in itertools.product((64, 33, 16, 8, 5, 2, 1), (width * 64, 1536, 300, 1), (None, 4096)):
        call.batch.n_seqs, call.batch.rows, call.batch.max_new = seqs, seqs * new, new
        call.batch.max_len, call.batch.cu = max_len, cu
        rc, need = call.size(heads=32, top=top)
        assert rc == 0
        sizes[seqs, max_len, cu] = need

        def why(size):  # at an address that every call refuses, once the size is enough
            out = []
            for dtype in (0, 1, 2):
                call.q.dtype = call.out.dtype = dtype
                args = (C.byref(call.cache), C.byref(call.batch), C.byref(call.q), 32, 0.1)
                end = (4100, size, None)
                if top:
                    rc = call.L.gvdb_kv_attend_topk_device(*args, top, 1, 1, C.byref(call.out), None, None, *end)
                else:
                    rc = call.L.gvdb_kv_attend_device(*args, 1, C.byref(call.out), None, *end)
                assert rc == ARG
                out.append("aligned" if "aligned" in call.why() else "below" if "below" in call.why() else call.why())
            return out

        assert why(need) == ["aligned"] * 3
        if need:
            assert "below" in why(need - 1)
    if new == 1 and not top:
        assert sizes[64, 1536, None] == 0 < sizes[1, 1536, None]


def test_chosen_pages_go_whole_or_along_the_line(call):  # noqa: F811
    """No size takes chosen pages in parts of a row: the kernels have no code for it."""
    call.cache.kv_heads, seen = 1, set()
    path = C.c_uint32()
    for page, width, top, seqs, new, heads, cu in itertools.product((32, 1024), (4, 300, 60000), (1, 30, 300, 65536), (1, 3, 190, 5000), (1, 7),
                                                                    (1, 20, 65536), (None, 4096)):
        call.cache.page_size, call.batch.table_width, call.batch.table_stride = page, width, width
        call.batch.n_seqs, call.batch.rows, call.batch.cu = seqs, seqs * new, cu
        for dtype in (0, 2):
            assert call.L.gvdb_kv_attend_path(C.byref(call.cache), C.byref(call.batch), dtype, heads, top, C.byref(path)) == 0
            seen.add(path.value)
    assert seen == {0, 2}
    for bad in ((3, 4, 1), (0, 0, 1), (0, 4, 65537)):
        assert call.L.gvdb_kv_attend_path(C.byref(call.cache), C.byref(call.batch), *bad, C.byref(path)) == ARG
    assert call.L.gvdb_kv_attend_path(C.byref(call.cache), C.byref(call.batch), 0, 4, 1, None) == ARG


@pytest.mark.parametrize("rows,heads,width", [(2048, 8, 32768), (100000, 8, 15361), (5000, 1, 100000), (3, 4096, 20000), (1, 64, 1 << 20)])
def test_scratch_of_long_tables_has_a_bound(call, rows, heads, width):  # noqa: F811
    """Page scores in scratch are those of one row, or 64 MiB; what else there is are the chosen pages and the parts of a join."""
    call.cache.kv_heads, call.batch.table_width, call.batch.table_stride = heads, width, width
    call.batch.n_seqs, call.batch.rows, call.batch.max_len = 1, rows, 4096
    rc, need = call.size(heads=heads, top=4)
    chosen, join = rows * heads * 4 * 4, 0
    path = C.c_uint32()
    for dtype in (0, 2):
        assert call.L.gvdb_kv_attend_path(C.byref(call.cache), C.byref(call.batch), dtype, heads, 4, C.byref(path)) == 0
        join |= path.value
    assert rc == 0 and need <= max(64 << 20, heads * width * 4) + chosen + (32 << 20 if join else 0) + 4096


# ---- the Python class, on CPU tensors and a library that only says yes ------------------------
class Kept(torch.Tensor):
    """A tensor that notes the streams that its memory is kept for."""

    def record_stream(self, stream):
        self.__dict__.setdefault("streams", []).append(stream)


@pytest.fixture()
def cache(gvdb_mod, monkeypatch):
    from contextlib import contextmanager
    from types import SimpleNamespace

    from gvdb import _ffi, kv

    now = ["here"]

    @contextmanager
    def stream(s):
        before, now[0] = now[0], s
        yield
        now[0] = before

    cuda = SimpleNamespace(current_stream=lambda dev: now[0], ExternalStream=lambda s, device: s, default_stream=lambda dev: "default", stream=stream)
    c = kv.KvCache.__new__(kv.KvCache)
    c.pool, c.bounds, c.bound_exps = (torch.zeros(n, dtype=torch.uint8).as_subclass(Kept) for n in (34 * 64 * 8, 64, 4))
    c.n_pages, c.kv_heads, c.head_dim, c.page_size, c.device = 4, 2, 64, 32, torch.device("cpu")
    c._torch = SimpleNamespace(cuda=cuda, empty=lambda *a, **k: torch.empty(*a, **k).as_subclass(Kept), uint8=torch.uint8, int32=torch.int32,
                               empty_like=lambda x: torch.empty_like(x).as_subclass(Kept), full=lambda *a, **k: torch.full(*a, **k).as_subclass(Kept),
                               bfloat16=torch.bfloat16, float32=torch.float32, is_grad_enabled=torch.is_grad_enabled)
    c._codes = {torch.float32: _ffi.GVDB_F32, torch.float16: _ffi.GVDB_F16, torch.bfloat16: _ffi.GVDB_BF16}
    c._i32, c._index, c._scale, c._sizes, c._ref = torch.int32, -1, 0.125, {}, None
    c.ran = []
    c._raw_stream = lambda index: c.ran.append(now[0])

    class Yes:
        def __getattr__(self, name):
            return lambda *a: 0

    c._lib = Yes()
    return c


def calls(cache):
    """Every call of the class, and the tensors that it is given."""
    def t(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype).as_subclass(Kept)

    q, k, v, table, lens, cu = t(3, 4, 64), t(3, 2, 64), t(3, 2, 64), t(2, 2, dtype=torch.int32), t(2, dtype=torch.int32), t(3, dtype=torch.int32)
    out, kv2, lse, chosen = t(3, 4, 64), (t(3, 2, 64), t(3, 2, 64)), t(3, 4), t(3, 2, 2, dtype=torch.int32)
    return [
        (lambda **s: cache.append(k, v, table, lens, cu=cu, **s), (k, v, table, lens, cu)),
        (lambda **s: cache.read(table, lens, 3, cu=cu, **s), (table, lens, cu)),
        (lambda **s: cache.read(table, lens, 3, cu=cu, out=kv2, **s), (table, lens, cu, *kv2)),
        (lambda **s: cache.attend(q, table, lens, cu=cu, **s), (q, table, lens, cu)),
        (lambda **s: cache.attend(q, table, lens, cu=cu, out=out, lse=lse, **s), (q, table, lens, cu, out, lse)),
        (lambda **s: cache.attend_topk(q, table, lens, 2, cu=cu, **s), (q, table, lens, cu)),
        (lambda **s: cache.attend_topk(q, table, lens, 2, cu=cu, out=out, chosen=chosen, lse=lse, **s), (q, table, lens, cu, out, chosen, lse)),
    ]


@pytest.mark.parametrize("number", range(7))
@pytest.mark.parametrize("stream,name", [(4242, 4242), (0, "default")])
def test_a_call_on_another_stream_keeps_what_it_works_on(cache, number, stream, name):
    """Dropped tensors would be handed out again on their own stream while the other one still reads or writes them."""
    run, given = calls(cache)[number]
    result = run(stream=stream)
    assert cache.ran == [name]
    for x in (*given, cache.pool, cache.bounds, cache.bound_exps):
        assert name in x.streams
    for x in () if result is None else result if isinstance(result, tuple) else (result,):
        assert "here" in x.streams
    run, given = calls(cache)[number]
    run()  # on the current stream nothing is noted
    assert cache.ran == [name, "here"] and not any(hasattr(x, "streams") for x in given)


def test_rows_that_require_a_gradient_are_refused(cache):
    """There is none to give: without a refusal training would go on with what the cache answered as a constant."""
    from gvdb import InvalidArgument

    table, lens = torch.zeros(2, 2, dtype=torch.int32).as_subclass(Kept), torch.zeros(2, dtype=torch.int32).as_subclass(Kept)
    q, kv = torch.zeros(2, 4, 64).as_subclass(Kept), torch.zeros(2, 2, 64).as_subclass(Kept)
    leaf, leaf_kv = q.clone().requires_grad_(), kv.clone().requires_grad_()
    for rows, other in ((leaf, leaf_kv), (leaf * 2, leaf_kv.transpose(0, 1).contiguous().transpose(0, 1))):
        tries = (lambda: cache.append(other, kv, table, lens), lambda: cache.append(kv, other, table, lens),
                 lambda: cache.read(table, lens, 2, out=(kv, other)), lambda: cache.attend(rows, table, lens),
                 lambda: cache.attend(q, table, lens, out=rows), lambda: cache.attend_topk(rows, table, lens, 2),
                 lambda: cache.attend(rows, table, lens, stream=7))
        for call_it in tries:
            with pytest.raises(InvalidArgument, match="gradient"):
                call_it()
            with torch.no_grad():
                call_it()
        cache.attend(rows.detach(), table, lens)
    assert not cache.attend(q, table, lens).requires_grad


def test_scales_beyond_the_range_of_floats(call):  # noqa: F811
    """In units of base 2, in which the kernels have it, a scale is finite too."""
    call.batch.table_width = call.batch.table_stride = 5000
    need = call.size()[1]
    for scale, why in ((2.3e38, "scratch"), (-2.3e38, "scratch"), (2.4e38, "scale"), (-3.4e38, "scale")):
        assert call.attend(scale=scale, size=need - 1) == ARG and why in call.why(), scale


@pytest.mark.parametrize("kind", ["tuple", "list", "stacked"])
def test_outputs_of_read_in_any_pair(cache, kind):
    table, lens = (torch.zeros(*s, dtype=torch.int32).as_subclass(Kept) for s in ((2, 2), (2,)))
    both = torch.zeros(2, 3, 2, 64).as_subclass(Kept)
    out = both if kind == "stacked" else (tuple if kind == "tuple" else list)(x.clone().as_subclass(Kept) for x in both)
    for stream in (None, 4242):
        assert cache.read(table, lens, 3, cu=torch.zeros(3, dtype=torch.int32).as_subclass(Kept), out=out, stream=stream) is out
