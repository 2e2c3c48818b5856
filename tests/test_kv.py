"""CPU: the token cache's plain form agrees with itself, and the C ABI refuses what it cannot do (no HIP call is made)."""
import ctypes as C

import numpy as np
import pytest

import kv_plain as plain


def test_quantise_ties_and_range():
    y = np.zeros((1, 32))
    y[0, :16] = [6.0, 5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 0.26, 5.01, 3.49, 2.49, 1.76, 1.24, 0.74, -6.0]
    got = plain.stored(y)[0, :16]
    assert got.tolist() == [6, 4, 4, 2, 2, 1, 1, 0, 0.5, 6, 3, 2, 2, 1, 0.5, -6]
    # just below 7 the largest stays under half a step off; at 7 the scale doubles
    for top, want in ((6.999, 6.0), (7.0, 8.0), (11.9, 12.0)):
        y[:] = 0
        y[0, 3] = top
        assert plain.stored(y)[0, 3] == want
    x = np.random.default_rng(0).standard_normal((1000, 128))
    k = plain.stored(x)
    g = np.abs(x.reshape(1000, 4, 32)).max(-1, keepdims=True)
    # half of the largest step (2) at the smallest scale ratio: amax >= 3.5 * 2^e
    assert (np.abs(k - x).reshape(1000, 4, 32) <= g / 3.5).all()


def test_bounds_hold():
    x = plain.stored(np.random.default_rng(1).standard_normal((40, 64)) * 3)
    b8, e = plain.bounds(x)
    s = 2.0 ** (e - 133)
    assert (b8[0] * s >= x.max(0)).all() and (b8[1] * s <= x.min(0)).all()
    assert np.abs(b8).max() <= 127 and np.abs(b8).max() >= 63


ARG = 6  # GVDB_ERR_INVALID_ARGUMENT


@pytest.fixture()
def call(gvdb_mod):
    """Structs of a call that is in order, on addresses that no refused call follows."""
    from gvdb import _ffi

    class Call:
        L = gvdb_mod.lib()
        cache = _ffi.gvdb_kv_cache(4096, 4096, 4096, 10, 2, 128, 64, 0)
        batch = _ffi.gvdb_kv_batch(4096, 5, 5, 2, 4096, None, 4, 0, 0, 0)
        rows = _ffi.gvdb_kv_rows(4096, 256, 128, 2, 0)
        q = _ffi.gvdb_kv_rows(4096, 512, 128, 2, 0)
        out = _ffi.gvdb_kv_rows(4096, 512, 128, 2, 0)

        def append(self):
            return self.L.gvdb_kv_append_device(C.byref(self.cache), C.byref(self.batch), C.byref(self.rows), C.byref(self.rows), None)

        def size(self, heads=4, top=0):
            n = C.c_uint64()
            return self.L.gvdb_kv_scratch_bytes(C.byref(self.cache), C.byref(self.batch), heads, top, C.byref(n)), n.value

        def attend(self, heads=4, scale=0.1, scratch=4096, size=1 << 40):
            return self.L.gvdb_kv_attend_device(C.byref(self.cache), C.byref(self.batch), C.byref(self.q), heads, scale, 1,
                                                C.byref(self.out), None, scratch, size, None)

        def topk(self, top=4, first=1, recent=1, scratch=4096, size=1 << 40):
            return self.L.gvdb_kv_attend_topk_device(C.byref(self.cache), C.byref(self.batch), C.byref(self.q), 4, 0.1, top, first,
                                                     recent, C.byref(self.out), None, None, scratch, size, None)

        def why(self):
            return self.L.gvdb_last_error().decode()

    # a call gets structs of its own
    Call.cache, Call.batch = (type(x).from_buffer_copy(x) for x in (Call.cache, Call.batch))
    return Call()


@pytest.mark.parametrize("field,value,code", [
    ("head_dim", 96, 3), ("head_dim", 0, 3), ("head_dim", 512, 3), ("page_size", 0, ARG), ("page_size", 48, ARG), ("page_size", 2048, ARG),
    ("kv_heads", 0, ARG), ("kv_heads", 5000, ARG), ("n_pages", 0, ARG), ("n_pages", 1 << 40, ARG), ("device", -1, ARG), ("pool", None, ARG),
    ("bounds", None, ARG), ("bound_exps", None, ARG), ("pool", 4097, ARG), ("bounds", 4104, ARG)])
def test_cache_refusals(call, field, value, code):
    setattr(call.cache, field, value)
    assert call.append() == code and call.why()
    assert call.attend() == code
    assert call.topk() == code
    assert call.size()[0] == code


@pytest.mark.parametrize("field,value", [
    ("n_seqs", 0), ("page_table", None), ("lengths", None), ("table_width", 0), ("table_width", 1 << 31), ("table_stride", 4),
    ("rows", 1 << 31), ("rows", 5)])
def test_batch_refusals(call, field, value):
    setattr(call.batch, field, value)
    assert call.append() == ARG and "token cache" in call.why()
    assert call.attend() == ARG
    assert call.topk() == ARG


def test_row_refusals(call):
    from gvdb import _ffi

    for field, value in (("data", None), ("dtype", 3), ("data", 4097), ("flags", 2)):
        keep = getattr(call.rows, field)
        setattr(call.rows, field, value)
        assert call.append() == ARG and call.why()
        setattr(call.rows, field, keep)
        keep = getattr(call.q, field)
        setattr(call.q, field, value)
        assert call.attend() == ARG
        setattr(call.q, field, keep)
    call.out.dtype = _ffi.GVDB_F32
    assert call.attend() == ARG and "one dtype" in call.why()
    call.out.dtype = _ffi.GVDB_BF16
    v = _ffi.gvdb_kv_rows(4096, 256, 128, 1, 0)
    assert call.L.gvdb_kv_append_device(C.byref(call.cache), C.byref(call.batch), C.byref(call.rows), C.byref(v), None) == ARG
    assert call.L.gvdb_kv_read_device(C.byref(call.cache), C.byref(call.batch), C.byref(call.rows), C.byref(v), None) == ARG


@pytest.mark.parametrize("field,value", [("row_stride", 0), ("row_stride", 127), ("row_stride", -127), ("head_stride", 0), ("head_stride", 64)])
def test_outputs_do_not_overlap(call, field, value):
    setattr(call.out, field, value)
    assert call.attend() == ARG and "overlapping" in call.why()
    assert call.topk() == ARG and "overlapping" in call.why()
    setattr(call.rows, field, value)
    for k, v in ((call.rows, None), (None, call.rows)):
        rc = call.L.gvdb_kv_read_device(C.byref(call.cache), C.byref(call.batch), k and C.byref(k), v and C.byref(v), None)
        assert rc == ARG and "overlapping" in call.why()


def test_attention_refusals(call):
    assert call.attend(heads=5) == ARG
    assert call.attend(heads=0) == ARG
    for scale in (float("nan"), float("inf")):
        assert call.attend(scale=scale) == ARG
    assert call.topk(top=0) == ARG
    assert call.topk(top=3, first=2, recent=2) == ARG
    call.batch.table_width = call.batch.table_stride = 5000
    rc, n = call.size()
    assert rc == 0 and n > 0
    assert call.attend(size=n - 1) == ARG and "scratch" in call.why()
    assert call.attend(scratch=None, size=n) == ARG
    assert call.attend(scratch=4100, size=n) == ARG
    rc, n = call.size(top=4)
    assert rc == 0 and call.topk(size=n - 1) == ARG


def test_nothing_to_do(call):
    call.batch.rows = 0
    assert call.append() == 0
    assert call.attend() == 0
    assert call.topk() == 0
    assert call.size() == (0, 0)


def test_scratch_is_a_rule_on_sizes(call):
    """Hints and sizes alone decide it: the same call asks for the same scratch."""
    call.batch.table_width = call.batch.table_stride = 5000
    a = call.size()
    assert a == call.size()
    call.batch.max_len = 64
    assert call.size()[1] <= a[1]
