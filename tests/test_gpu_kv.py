"""GPU: the token cache's operators against their definition in 64 bits."""
import numpy as np
import pytest
import torch

import kv_plain as plain

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}   # a rounding is off by at most this, relatively
TINY = {"bf16": 2.0 ** -133, "f16": 2.0 ** -25, "f32": 2.0 ** -149}  # ... or this, below the normal range
PROB = {"bf16": 2.0 ** -8, "f16": 2.0 ** -16, "f32": 2.0 ** -24}   # the probabilities' bits


@pytest.fixture()
def kv(gvdb_mod):
    from gvdb import kv

    return kv


class Store:
    """A cache filled through append, and the stored values in 64 bits.  Whatever was not written reads as NaN."""

    def __init__(self, kv, seed, dtype, heads, D, page, lens, spread=1.0, width=None):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lens]
        self.width = width or max(1, max(need)) + 1
        self.n_pages = sum(need) + 2
        order = rng.permutation(self.n_pages)
        table = np.full((len(lens), self.width), -7, np.int32)
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.cache = kv.KvCache(self.n_pages, heads, D, page)
        self.cache.pool.fill_(255)
        self.cache.bounds.fill_(-1)
        self.cache.bound_exps.fill_(255)
        self.table = torch.from_numpy(table).cuda()
        self.lens, self.page, self.heads, self.D, self.dtype = list(lens), page, heads, D, dtype
        self.k, self.v = [], []
        rows_k, rows_v = [], []
        for n in lens:
            k = rng.standard_normal((n, heads, D)) + rng.standard_normal((1, heads, D))
            k[:, :, : D // 16] *= 4
            k += 0.7 * np.repeat(rng.standard_normal((n // 16 + 1, heads, D)), 16, 0)[:n]
            rows_k.append(torch.from_numpy(k * spread).to(DT[dtype]))
            rows_v.append(torch.from_numpy(rng.standard_normal((n, heads, D))).to(DT[dtype]))
        self.cu = torch.from_numpy(np.cumsum([0] + list(lens)).astype(np.int32)).cuda()
        k, v = torch.cat(rows_k), torch.cat(rows_v)
        if len(k):
            self.cache.append(k.cuda(), v.cuda(), self.table, self.zeros(), cu=self.cu)
        for a, b in zip(rows_k, rows_v):
            self.k.append(plain.stored(a.double().numpy()))
            self.v.append(plain.stored(b.double().numpy()))

    def zeros(self):
        return torch.zeros(len(self.lens), dtype=torch.int32, device="cuda")

    def lengths(self):
        return torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    def bounds(self, s, h):
        n, P = self.lens[s], self.page
        return [plain.bounds(self.k[s][p:min(p + P, n), h]) for p in range(0, n, P)]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def queries(seed, dtype, new, heads, D):
    rng = np.random.default_rng(seed)
    return torch.from_numpy(rng.standard_normal((sum(new), heads, D))).to(DT[dtype])


def check_attend(st, q, new, out, lse=None, causal=True, scale=None, chosen=None, skip=()):
    """Every output within its bound: the output's rounding, the probabilities' bits, and 32-bit sums of scores and products."""
    D, dtype = st.D, st.dtype
    scale = D ** -0.5 if scale is None else scale
    Hq = q.shape[1]
    g = Hq // st.heads
    out = out.double().cpu().numpy()
    qd = q.double().cpu().numpy()
    row = 0
    for s, n in enumerate(new):
        L = st.lens[s]
        for i in range(n):
            for hq in range(Hq):
                if (row, hq) in skip:
                    continue
                h = hq // g
                sees = np.arange(L) < (L - n + i + 1 if causal else L)
                if chosen is not None:
                    mine = np.isin(np.arange(L) // st.page, chosen[row, h][chosen[row, h] >= 0])
                    sees &= mine
                o, ls, absum, s1 = plain.attend(qd[row, hq], st.k[s][:, h], st.v[s][:, h], scale, sees)
                # a score is off by (D + 8) roundings of its terms' sum, a sum of n terms by n / 32 + 64 roundings
                rel = 2 * (D + 8) * 2.0 ** -24 * s1 + (L / 32 + 64) * 2.0 ** -23
                tol = HALF[dtype] * np.abs(o) + (PROB[dtype] + rel) * (1 + HALF[dtype]) * absum + TINY[dtype]
                err = np.abs(out[row, hq] - o)
                assert (err <= tol).all(), (s, i, hq, float((err / np.maximum(tol, 1e-300)).max()))
                if lse is not None:
                    got = float(lse[row, hq])
                    assert got == ls if np.isinf(ls) else abs(got - ls) <= rel + 2.0 ** -22 * (abs(ls) + 8), (s, i, hq, got, ls)
            row += 1


# ---- append and read ----------------------------------------------------------------------
@pytest.mark.parametrize("dtype,heads,D,page,lens", [
    ("bf16", 2, 128, 64, (1, 63, 64, 65, 200)),
    ("f32", 3, 64, 32, (31, 0, 97, 1)),
    ("f16", 1, 256, 128, (130, 5)),
    ("f32", 2, 128, 96, (300,)),
])
def test_append_stores_what_it_should(kv, dtype, heads, D, page, lens):
    st = Store(kv, 1, dtype, heads, D, page, lens)
    k, v = st.cache.read(st.table, st.zeros(), sum(lens), cu=st.cu, dtype=torch.float32)
    k, v = k.double().cpu().numpy(), v.double().cpu().numpy()
    assert np.array_equal(k, np.concatenate(st.k)) and np.array_equal(v, np.concatenate(st.v))
    # the buffers are laid out as documented
    pool, b8, be = st.cache.pool.cpu().numpy(), st.cache.bounds.cpu().numpy(), st.cache.bound_exps.cpu().numpy()
    table = st.table.cpu().numpy()
    used = set()
    for s, n in enumerate(lens):
        for h in range(heads):
            for j, want in enumerate(st.bounds(s, h)):
                pg = table[s, j]
                used.add(int(pg))
                assert np.array_equal(b8[pg, h], want[0]) and be[pg, h] == want[1]
                for t in range(0, min(page, n - j * page), 32):
                    a, b = plain.tile_values(pool[pg, h, t // 32], D)
                    m = min(32, n - j * page - t)
                    assert np.array_equal(a[:m], st.k[s][j * page + t:j * page + t + m, h])
                    assert np.array_equal(b[:m], st.v[s][j * page + t:j * page + t + m, h])
                    # what lies behind was left alone
                    assert np.isnan(a[m:]).all() and np.isnan(b[m:]).all()
    for pg in set(range(st.n_pages)) - used:
        assert (pool[pg] == 255).all() and (be[pg] == 255).all() and (b8[pg] == -1).all()


def test_append_in_pieces_is_append_at_once(kv):
    """Token by token, in runs over page borders, and written twice: the same bytes."""
    D, heads, page, n = 128, 2, 64, 200
    x = torch.randn(n, heads, D, dtype=torch.bfloat16, device="cuda")
    y = torch.randn(n, heads, D, dtype=torch.bfloat16, device="cuda")
    table = i32([[3, 0, 4, 2]])
    got = []
    for cuts in ([0, n], list(range(n + 1)), [0, 1, 63, 64, 130, n], [0, 150, n]):
        c = kv.KvCache(5, heads, D, page)
        c.pool.zero_(), c.bounds.zero_(), c.bound_exps.zero_()
        for a, b in zip(cuts, cuts[1:]):
            c.append(x[a:b], y[a:b], table, i32([a]))
        c.append(x[17:90], y[17:90], table, i32([17]), max_new=1) if cuts[1] == 150 else None
        if cuts[1] == 150:  # the rewrite ended inside a page: its bounds cover what it wrote up to there
            c.append(x[64:128], y[64:128], table, i32([64]))
        got.append((c.pool.clone(), c.bounds.clone(), c.bound_exps.clone()))
    for other in got[1:]:
        for a, b in zip(got[0], other):
            assert torch.equal(a, b)


def test_append_extremes(kv):
    """Zeros, the smallest and largest floats, ties, infinities and NaN."""
    D = 64
    rng = np.random.default_rng(5)
    x = rng.standard_normal((40, 1, D)).astype(np.float32)
    x[0] = 0
    x[1] = 1e-45
    x[2] *= 1e-38
    x[3] = 3.4028235e38
    x[4] *= 1e37
    x[5, 0, :32] = np.array([6, 5, 3.5, 2.5, 1.75, 1.25, .75, .25] * 4) * np.tile([1, -1], 16)
    x[6, 0, 32:] = np.array([7, 5, 3.5, 2.5, 1.75, 1.25, .75, .25] * 4)
    x[7, 0, 3] = np.inf
    x[8, 0, 40] = -np.inf
    x[9, 0, 10] = np.nan
    x[10, 0, 0] = np.float32(6.9999995)
    want = plain.stored(x.astype(np.float64))
    c = kv.KvCache(2, 1, D, 32)
    t = torch.from_numpy(x).cuda()
    c.append(t, t.flip(2), i32([[1, 0]]), i32([0]))
    k, v = c.read(i32([[1, 0]]), i32([0]), 40, dtype=torch.float32)
    assert np.array_equal(k.double().cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(v.flip(2).double().cpu().numpy()[10:], want[10:], equal_nan=True)
    assert c.bound_exps.cpu().tolist()[1] == [255] and c.bound_exps.cpu().tolist()[0] != [255]


def test_append_and_read_strided_and_misaligned(kv):
    D, heads = 128, 3
    base = torch.randn(50, 2 * heads + 1, D, device="cuda").to(torch.float16)
    k, v = base[:, :heads], base[:, heads:2 * heads]
    off = torch.randn(50 * heads * D + 3, device="cuda").to(torch.float16)[3:].view(50, heads, D)
    table = i32([[0, 1]])
    for a, b in ((k, v), (off, v), (k.flip(0).transpose(0, 1).contiguous().transpose(0, 1), off)):
        c = kv.KvCache(2, heads, D, 32)
        c.append(a, b, table, i32([0]))
        out = torch.full((2, 50, heads, 2 * D), 7.0, dtype=torch.float16, device="cuda")
        c.read(table, i32([0]), 50, out=(out[0, :, :, :D], out[1, :, :, 1:D + 1]))
        assert np.array_equal(out[0, :, :, :D].double().cpu().numpy(), plain.stored(a.double().cpu().numpy()))
        assert np.array_equal(out[1, :, :, 1:D + 1].double().cpu().numpy(), plain.stored(b.double().cpu().numpy()))
        assert (out[0, :, :, D:] == 7).all() and (out[1, :, :, 0] == 7).all() and (out[1, :, :, D + 1:] == 7).all()


def test_pages_that_are_not_there(kv):
    """No page number is followed out of the pool or the table: append skips, read and attention give NaN."""
    D, page = 64, 32
    x = torch.randn(3 * 96, 1, D, device="cuda")
    table = i32([[0, -1, 1], [2, 3, 99], [4, 5, 6]])
    c = kv.KvCache(7, 1, D, page)
    c.append(x, x, table, i32([0, 0, 0]))
    k, v = c.read(table, i32([0, 0, 0]), 288, dtype=torch.float32)
    k = k.view(3, 96, D)
    want = plain.stored(x.double().cpu().numpy()).reshape(3, 96, D)
    bad = np.zeros((3, 96), bool)
    bad[0, 32:64] = bad[1, 64:] = True
    assert torch.isnan(k).all(-1).squeeze().cpu().numpy().reshape(3, 96).tolist() == bad.tolist()
    assert np.array_equal(k.double().cpu().numpy()[~bad], want[~bad])
    q = torch.randn(6, 2, D, device="cuda")
    for lens, nan in (((33, 64, 96), (0,)), ((32, 65, 96), (1,)), ((32, 64, 97), (2,))):
        many = q.to(torch.bfloat16).view(3, 2, 2, D).repeat_interleave(40, 1).view(240, 2, D).contiguous()  # 160 rows a sequence
        wide = c.attend(many, table, i32(lens)).view(3, 80, 2, D)
        assert torch.isnan(wide[:, -1]).flatten(1).all(1).tolist() == [s in nan for s in range(3)]
        for o in (c.attend(q, table, i32(lens)), c.attend_topk(q, table, i32(lens), 3)[0]):
            got = torch.isnan(o).flatten(1).all(1).cpu().view(3, 2)[:, 1].nonzero().flatten().tolist()
            assert got == list(nan), (lens, got)
            fine = torch.isfinite(o).flatten(1).all(1).cpu().view(3, 2)
            assert all(fine[s, 1] for s in range(3) if s not in nan)


# ---- attention ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,Hq,heads,D,page,lens,new", [
    ("bf16", 8, 2, 128, 64, (1,), (1,)),
    ("bf16", 32, 8, 128, 64, (777, 0, 1, 64, 65, 1500), (1,) * 6),
    ("f16", 6, 2, 64, 32, (300, 33, 31), (1, 1, 1)),
    ("f32", 4, 4, 256, 128, (129, 500), (1, 1)),
    ("f32", 7, 1, 128, 32, (250,), (1,)),
    ("bf16", 40, 2, 64, 32, (100, 999), (1, 1)),          # more heads a group than a tile has rows
    ("f16", 4, 2, 128, 64, (40, 3, 130), (5, 5, 5)),      # a sequence shorter than its rows: the first see nothing
    ("bf16", 8, 2, 128, 64, (65, 300), (65, 37)),
    ("f32", 3, 1, 64, 96, (100, 0, 50), (100, 4, 50)),
    ("f16", 5, 5, 256, 32, (70, 41), (33, 41)),
    ("bf16", 12, 4, 64, 64, (260,), (131,)),
])
def test_attend(kv, dtype, Hq, heads, D, page, lens, new):
    st = Store(kv, 2, dtype, heads, D, page, lens)
    q = queries(3, dtype, new, Hq, D).cuda()
    cu = i32(np.cumsum((0,) + new).tolist())
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = st.cache.attend(q, st.table, st.lengths(), cu=cu, lse=lse, max_new=max(new), max_len=max(lens))
    check_attend(st, q, new, out, lse)
    if len(set(new)) == 1:  # without cu the keys may be cut elsewhere: another order of the same sums, under the same bound
        check_attend(st, q, new, st.cache.attend(q, st.table, st.lengths(), max_len=max(lens)))
    # hints size the launch only: too small, too large and none give the same sums, in another order
    for hints in ({"max_new": 1, "max_len": 1}, {}, {"max_new": 10 ** 6, "max_len": 10 ** 6}):
        check_attend(st, q, new, st.cache.attend(q, st.table, st.lengths(), cu=cu, **hints))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_without_causal_and_with_scale(kv, dtype):
    st = Store(kv, 4, dtype, 2, 128, 64, (90, 10, 0))
    new = (4, 20, 3)
    q = queries(5, dtype, new, 4, 128).cuda()
    cu = i32([0, 4, 24, 27])
    lse = torch.empty(27, 4, device="cuda")
    out = st.cache.attend(q, st.table, st.lengths(), cu=cu, causal=False, scale=-0.3, lse=lse)
    check_attend(st, q, new, out, lse, causal=False, scale=-0.3)


@pytest.mark.parametrize("dtype,lens", [("bf16", (9000, 4001)), ("f16", (20000,)), ("f32", (6001, 5, 7777))])
def test_attend_split_along_the_keys(kv, dtype, lens):
    """Few rows and long contexts: the parts are joined by a second kernel, alike on every run."""
    st = Store(kv, 6, dtype, 2, 128, 64, lens)
    q = queries(7, dtype, (1,) * len(lens), 6, 128).cuda()
    lse = torch.empty(len(lens), 6, device="cuda")
    out = st.cache.attend(q, st.table, st.lengths(), lse=lse)
    check_attend(st, q, (1,) * len(lens), out, lse)
    for _ in range(3):
        assert torch.equal(out, st.cache.attend(q, st.table, st.lengths()))


@pytest.mark.parametrize("dtype,spread", [("bf16", 30.0), ("f32", 30.0), ("f16", 1e-3)])
def test_attend_sharp_and_flat(kv, dtype, spread):
    st = Store(kv, 8, dtype, 1, 64, 32, (500,), spread)
    q = queries(9, dtype, (3,), 4, 64).cuda()
    check_attend(st, q, (3,), st.cache.attend(q, st.table, st.lengths()))


@pytest.mark.parametrize("dtype,heads,Hq,D,page", [("f32", 1, 2, 128, 64), ("bf16", 1, 2, 128, 64), ("f16", 1, 2, 64, 32), ("bf16", 2, 4, 256, 96)])
def test_what_is_masked_may_hold_anything(kv, dtype, heads, Hq, D, page):
    """A key or value that is not finite shows in the rows that see it, and in no other; a value only in its group of channels."""
    for poison in (float("nan"), float("inf"), -float("inf")):
        st = Store(kv, 10, dtype, heads, D, page, (150,))
        k = torch.from_numpy(np.random.default_rng(1).standard_normal((4, heads, D))).to(DT[dtype]).cuda()
        v = k.clone()
        v[1, :, 40] = poison   # token 121: a value, channels 32 .. 63
        k[3, :, 7] = poison    # token 123: a key
        st.cache.append(k, v, st.table, i32([120]))
        st.k[0][120:124], st.v[0][120:124] = plain.stored(k.double().cpu().numpy()), plain.stored(v.double().cpu().numpy())
        q = queries(11, dtype, (150,), Hq, D).cuda()
        lse = torch.empty(150, Hq, device="cuda")
        out = st.cache.attend(q, st.table, st.lengths(), lse=lse)
        nan = torch.isnan(out).cpu().numpy()
        want = np.zeros((150, Hq, D), bool)
        want[121:, :, 32:64] = True
        want[123:] = True
        assert np.array_equal(nan, want)
        skip = {(r, h) for r in range(121, 150) for h in range(Hq)}
        check_attend(st, q, (150,), out, skip=skip)
        # the channels beside the value's group are what they would be
        got = out.double().cpu().numpy()[121:123]
        for r in range(2):
            for hq in range(Hq):
                h = hq // (Hq // heads)
                n = 122 + r
                vv = np.nan_to_num(st.v[0][:n, h])
                o, _, absum, _ = plain.attend(q[121 + r, hq].double().cpu().numpy(), st.k[0][:n, h], vv, D ** -0.5, np.ones(n, bool))
                other = np.r_[0:32, 64:D]
                assert (np.abs(got[r, hq] - o)[other] <= (HALF[dtype] * np.abs(o) + 2 * (PROB[dtype] + 2.0 ** -12) * absum)[other]).all()
        # single tokens over a shorter length
        for n, bad in ((121, False), (122, True), (124, True)):
            one = st.cache.attend(q[:1], st.table, i32([n]))
            assert bool(torch.isnan(one).any()) == bad
            assert bool(torch.isnan(one).all()) == (n == 124)


def test_a_query_that_is_not_finite_spoils_its_own_row(kv):
    for new, Hq in (((2, 2), 4), ((70, 66), 4)):
        st = Store(kv, 12, "bf16", 2, 64, 32, (80, 80))
        q = queries(13, "bf16", new, Hq, 64).cuda()
        q[1, 2, 5] = float("nan")
        q[new[0], 0, 0] = float("inf")
        out = st.cache.attend(q, st.table, st.lengths(), cu=i32([0, new[0], sum(new)]))
        assert torch.isnan(out[1, 2]).all() and torch.isnan(out[new[0], 0]).all()
        check_attend(st, q, new, out, skip={(1, 2), (new[0], 0)})


@pytest.mark.parametrize("dtype,Hq,heads,D,page,lens,new,causal", [
    ("bf16", 8, 2, 64, 32, (400, 70, 9), (33, 70, 40), True),     # the last sequence is shorter than its rows
    ("f16", 8, 2, 128, 64, (500, 0), (200, 3), False),
    ("bf16", 4, 2, 256, 64, (300,), (129,), True),
    ("f16", 3, 1, 256, 1024, (1300,), (47,), True),
    ("bf16", 64, 1, 64, 64, (4000,), (5,), True),                 # few rows blocks: split along the keys
    ("f16", 32, 2, 128, 96, (3000, 2500), (8, 9), True),
])
def test_attend_many_rows(kv, dtype, Hq, heads, D, page, lens, new, causal):
    st = Store(kv, 40, dtype, heads, D, page, lens)
    q = queries(41, dtype, new, Hq, D).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    out = st.cache.attend(q, st.table, st.lengths(), cu=i32(np.cumsum((0,) + new).tolist()), causal=causal, lse=lse, max_new=max(new))
    check_attend(st, q, new, out, lse, causal=causal)


def crowd(st, q, new, copies, lse=None, **more):
    """The same sequences many times over, as many as take whole workgroups of rows: every copy's output is the first's."""
    rows = len(q)
    many = torch.empty(rows * copies, q.shape[1], device="cuda")
    out = st.cache.attend(q.repeat(copies, 1, 1), st.table.repeat(copies, 1), st.lengths().repeat(copies),
                          cu=i32(np.cumsum((0,) + tuple(new) * copies).tolist()), lse=many, max_new=max(new), **more)
    bits = out.view(torch.int16 if out.element_size() == 2 else torch.int32).view(copies, rows, *q.shape[1:])
    assert torch.equal(bits, bits[:1].expand_as(bits))
    if lse is not None:
        lse.copy_(many[:rows])
    return out[:rows]


@pytest.mark.parametrize("dtype,Hq,heads,D,page,lens,new,causal,copies", [
    ("bf16", 8, 2, 64, 32, (400, 70, 9), (33, 70, 40), True, 60),     # the last sequence is shorter than its rows
    ("f16", 8, 2, 64, 32, (130, 77), (64, 40), False, 60),
    ("f16", 8, 2, 128, 64, (500, 0), (200, 3), False, 30),
    ("bf16", 6, 2, 128, 64, (333,), (90,), True, 60),
    ("bf16", 4, 2, 256, 64, (300,), (129,), True, 64),
    ("f16", 3, 1, 256, 1024, (1000,), (47,), True, 128),
    ("bf16", 8, 1, 64, 32, (400,), (128,), True, 96),                 # rows that fill whole workgroups
    ("f16", 8, 1, 64, 64, (390,), (127,), False, 96),
    ("bf16", 8, 1, 128, 96, (400,), (128,), True, 96),
    ("f16", 8, 1, 128, 32, (399,), (127,), True, 96),
    ("bf16", 8, 1, 256, 64, (400,), (128,), True, 96),
    ("f16", 8, 1, 256, 1024, (393,), (128,), False, 96),
])
def test_attend_crowds_of_rows(kv, dtype, Hq, heads, D, page, lens, new, causal, copies):
    st = Store(kv, 45, dtype, heads, D, page, lens)
    q = queries(46, dtype, new, Hq, D).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    check_attend(st, q, new, crowd(st, q, new, copies, lse, causal=causal, max_len=max(lens)), lse, causal=causal)


@pytest.mark.parametrize("dtype,Hq,heads,D,lens,new", [("bf16", 64, 1, 64, (4000,), (5,)), ("f16", 32, 2, 128, (3000, 2500), (8, 9)),
                                                       ("bf16", 16, 1, 256, (1500,), (9,)), ("bf16", 64, 1, 64, (3000, 2500), (16, 15)),
                                                       ("f16", 64, 1, 128, (3000, 2500), (16, 15)), ("f16", 64, 1, 256, (2600, 400), (16, 15))])
def test_attend_many_rows_in_parts(kv, dtype, Hq, heads, D, lens, new):
    """A table far wider than the sequences: parts are cut for the width, and most of them hold nothing."""
    st = Store(kv, 47, dtype, heads, D, 64, lens, width=4000)
    q = queries(48, dtype, new, Hq, D).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    out = st.cache.attend(q, st.table, st.lengths(), cu=i32(np.cumsum((0,) + new).tolist()), lse=lse, max_new=max(new))
    every = [(i, h) for i in range(len(q)) for h in range(Hq)]
    check_attend(st, q, new, out, lse, skip=set(every) - set(every[::5]))


@pytest.mark.parametrize("dtype,Hq,heads,D,lens,new", [("bf16", 32, 1, 64, (12000, 11000), 64), ("f16", 32, 1, 128, (12000, 11000), 64),
                                                       ("f16", 32, 1, 256, (12000, 11000), 64), ("bf16", 32, 1, 128, (12000, 11000), 63),
                                                       ("bf16", 32, 2, 64, (12500,), 32), ("f16", 16, 2, 128, (7000, 6500), 64),
                                                       ("bf16", 16, 1, 256, (12400,), 64), ("f16", 24, 3, 64, (3300, 5000, 17, 0), 70)])
def test_attend_many_rows_in_rounds(kv, dtype, Hq, heads, D, lens, new):
    """As many rows each sequence: parts by rounds of workgroups.  Every 97th row and head is checked."""
    st = Store(kv, 53, dtype, heads, D, 64, lens)
    q = queries(54, dtype, (new,) * len(lens), Hq, D).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    every = [(i, h) for i in range(len(q)) for h in range(Hq)]
    for hints in ({"max_len": max(lens)}, {}, {"max_len": 500}):
        out = st.cache.attend(q, st.table, st.lengths(), lse=lse, **hints)
        check_attend(st, q, (new,) * len(lens), out, lse, skip=set(every) - set(every[::97]))


@pytest.mark.parametrize("dtype,Hq,D,page,copies", [("bf16", 4, 128, 64, 96), ("f16", 4, 64, 32, 96), ("bf16", 4, 256, 96, 48),
                                                    ("f16", 4, 128, 32, 96), ("bf16", 2, 64, 32, 96)])
def test_what_is_masked_in_a_crowd_may_hold_anything(kv, dtype, Hq, D, page, copies):
    for poison in (float("nan"), float("inf"), -float("inf")):
        st = Store(kv, 49, dtype, 1, D, page, (150,))
        k = torch.from_numpy(np.random.default_rng(1).standard_normal((4, 1, D))).to(DT[dtype]).cuda()
        v = k.clone()
        v[1, :, 40] = poison   # token 121: a value, channels 32 .. 63
        k[3, :, 7] = poison    # token 123: a key
        st.cache.append(k, v, st.table, i32([120]))
        st.k[0][120:124], st.v[0][120:124] = plain.stored(k.double().cpu().numpy()), plain.stored(v.double().cpu().numpy())
        q = queries(50, dtype, (150,), Hq, D).cuda()
        q[5, 1, 0] = poison
        out = crowd(st, q, (150,), copies, max_len=150)
        want = np.zeros((150, Hq, D), bool)
        want[121:, :, 32:64] = True
        want[123:] = True
        want[5, 1] = True
        assert np.array_equal(torch.isnan(out).cpu().numpy(), want)
        check_attend(st, q, (150,), out, skip={(r, h) for r in range(121, 150) for h in range(Hq)} | {(5, 1)})
        table = st.table.clone()
        table[0, 1] = -1       # a page that is not there
        st.table = table
        nan = torch.isnan(crowd(st, q, (150,), copies, max_len=150)).flatten(1).all(1)
        assert nan.tolist() == [r >= page for r in range(150)]


def test_rows_outside_every_sequence(kv):
    """cu may begin behind the first row and end before the last: those rows are left alone, or 0 where the call makes the output."""
    D, Hq, heads = 64, 4, 2
    for new, dtype in (((3, 2), "f32"), ((70, 40), "bf16")):
        st = Store(kv, 42, dtype, heads, D, 32, (100, 90))
        q = queries(43, dtype, (2 + sum(new) + 3,), Hq, D).cuda()
        cu = i32([2, 2 + new[0], 2 + sum(new)])
        rest = [0, 1] + list(range(2 + sum(new), 5 + sum(new)))
        for given in (False, True):
            keep = torch.full_like(q, 9.0) if given else None
            out = st.cache.attend(q, st.table, st.lengths(), cu=cu, out=keep)
            got, chosen = st.cache.attend_topk(q, st.table, st.lengths(), 2, cu=cu, out=keep.clone() if given else None)
            for o in (out, got):
                assert (o[rest] == (9 if given else 0)).all()
            assert (chosen[rest] == -1).all()
            check_attend(st, q[2:-3], new, out[2:-3])
            check_attend(st, q[2:-3], new, got[2:-3], chosen=chosen[2:-3].cpu().numpy())
        k, v = st.cache.read(st.table, st.zeros(), q.shape[0], cu=cu, dtype=torch.float32)
        assert (k[rest] == 0).all() and (v[rest] == 0).all() and torch.isfinite(k).all()
        assert np.array_equal(k[2:2 + new[0]].double().cpu().numpy(), st.k[0][:new[0]])


def test_pools_over_32_bits(kv):
    """Pages whose bytes lie behind 4 GiB."""
    D, heads, page, n = 256, 8, 64, 40000
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB")
    c = kv.KvCache(n, heads, D, page)
    assert c.pool.numel() > 5 << 30
    table = i32([[n - 1, 3, n - 7, 35000, 0]])
    x, y = (torch.randn(300, heads, D, device="cuda") for _ in range(2))
    c.append(x, y, table, i32([0]))
    k, v = c.read(table, i32([0]), 300, dtype=torch.float32)
    assert np.array_equal(k.double().cpu().numpy(), plain.stored(x.double().cpu().numpy()))
    assert np.array_equal(v.double().cpu().numpy(), plain.stored(y.double().cpu().numpy()))
    st = Store.__new__(Store)
    st.__dict__.update(cache=c, table=table, lens=[300], page=page, heads=heads, D=D, dtype="f32", k=[k.double().cpu().numpy()],
                       v=[v.double().cpu().numpy()])
    q = queries(44, "f32", (2,), heads, D).cuda()
    check_attend(st, q, (2,), c.attend(q, table, i32([300])))
    out, chosen = c.attend_topk(q, table, i32([300]), 3)
    check_attend(st, q, (2,), out, chosen=chosen.cpu().numpy())


def test_strided_misaligned_and_given_outputs(kv):
    D, Hq, heads = 128, 4, 2
    st = Store(kv, 14, "bf16", heads, D, 64, (100, 70))
    fused = torch.randn(10, Hq + 2 * heads, D, device="cuda").to(torch.bfloat16)
    new = (4, 3)
    cu = i32([0, 4, 7])  # rows 7 .. 9 belong to no sequence
    flat = torch.randn(10 * Hq * D + 1, device="cuda").to(torch.bfloat16)[1:].view(10, Hq, D)
    for q in (fused[:, :Hq], flat):
        big = torch.full((10, Hq, D + 5), 3.0, dtype=torch.bfloat16, device="cuda")
        lse = torch.full((10, Hq), 3.0, device="cuda")
        out = st.cache.attend(q, st.table, st.lengths(), cu=cu, out=big[:, :, 2:D + 2], lse=lse)
        check_attend(st, q, new, out, lse)
        assert (big[7:] == 3).all() and (big[:, :, :2] == 3).all() and (big[:, :, D + 2:] == 3).all() and (lse[7:] == 3).all()
        got, chosen = st.cache.attend_topk(q, st.table, st.lengths(), 4, cu=cu)
        check_attend(st, q, new, got, chosen=chosen.cpu().numpy())
        assert (got[7:] == 0).all() and (chosen[7:] == -1).all()


@pytest.mark.parametrize("dtype,new,lens", [("bf16", (2, 2), (9000, 4001)), ("f32", (3, 1), (5000, 2222)), ("f16", (90, 70), (3000, 700)),
                                            ("bf16", (5, 0), (7, 640))])
def test_hints_decide_nothing(kv, dtype, new, lens):
    """Hints far below and above the truth, with and without `cu`; and the queries' own memory for the output."""
    st = Store(kv, 40, dtype, 2, 64, 32, lens)
    q = queries(41, dtype, new, 4, 64).cuda()
    cu = i32(np.cumsum((0,) + new).tolist())
    for hints in ({"max_new": 1, "max_len": 1}, {"max_new": 3, "max_len": 100}, {"max_new": 4000000000, "max_len": 4000000000}):
        lse = torch.empty(q.shape[:2], device="cuda")
        check_attend(st, q, new, st.cache.attend(q, st.table, st.lengths(), cu=cu, lse=lse, **hints), lse)
        if new[0] == new[1]:
            check_attend(st, q, new, st.cache.attend(q, st.table, st.lengths(), **hints))
    for cus in [cu] + [None] * (new[0] == new[1]):
        want, own = st.cache.attend(q, st.table, st.lengths(), cu=cus), q.clone()
        assert st.cache.attend(own, st.table, st.lengths(), cu=cus, out=own) is own and torch.equal(own, want)
        (want, pages), own = st.cache.attend_topk(q, st.table, st.lengths(), 5, cu=cus), q.clone()
        _, again = st.cache.attend_topk(own, st.table, st.lengths(), 5, cu=cus, out=own)
        assert torch.equal(own, want) and torch.equal(again, pages)


# ---- attention over chosen pages --------------------------------------------------------------
@pytest.mark.parametrize("dtype,Hq,heads,D,page,lens,new,top,first,recent", [
    ("bf16", 8, 2, 128, 64, (5000,), (1,), 8, 1, 1),
    ("bf16", 32, 8, 128, 64, (3000, 0, 1, 64, 65, 2111), (1,) * 6, 6, 1, 2),
    ("f16", 6, 2, 64, 32, (900, 40), (3, 2), 5, 0, 0),
    ("f32", 5, 5, 256, 32, (700, 310), (1, 4), 4, 2, 2),
    ("f32", 20, 1, 64, 32, (600,), (2,), 7, 1, 1),
    ("bf16", 3, 1, 128, 128, (2000, 7, 30), (9, 7, 40), 3, 1, 1),
    ("f16", 4, 4, 128, 32, (500,), (40,), 100, 1, 1),     # more than there are: everything
    ("bf16", 4, 2, 64, 32, (300, 200), (1, 1), 1, 0, 1),
    ("f16", 4, 1, 256, 32, (600,), (20,), 5, 1, 1),       # prompts: several times 16 columns share the bounds
    ("f32", 14, 2, 64, 32, (900, 33), (21, 12), 6, 2, 1),
    ("bf16", 34, 2, 128, 32, (800,), (7,), 70, 1, 3),     # more heads a group than columns, more pages than a wave has lanes
])
def test_attend_topk(kv, dtype, Hq, heads, D, page, lens, new, top, first, recent):
    st = Store(kv, 15, dtype, heads, D, page, lens)
    q = queries(16, dtype, new, Hq, D).cuda()
    cu = i32(np.cumsum((0,) + new).tolist())
    lse = torch.empty(q.shape[:2], device="cuda")
    out, chosen = st.cache.attend_topk(q, st.table, st.lengths(), top, first=first, recent=recent, cu=cu, lse=lse, max_new=max(new),
                                       max_len=max(lens))
    got = chosen.cpu().numpy()
    qd = q.double().cpu().numpy()
    g = Hq // heads
    row = 0
    for s, n in enumerate(new):
        bounds = [st.bounds(s, h) for h in range(heads)]
        for i in range(n):
            place = lens[s] - n + i
            seen = place // page + 1 if place >= 0 else 0
            for h in range(heads):
                want = plain.choose(qd[row, h * g:(h + 1) * g], bounds[h], seen, top, first, recent)
                assert got[row, h].tolist() == want + [-1] * (top - len(want)), (s, i, h)
            row += 1
    check_attend(st, q, new, out, lse, chosen=got)
    for hints in ({"max_new": 1, "max_len": 1}, {}):
        o2, c2 = st.cache.attend_topk(q, st.table, st.lengths(), top, first=first, recent=recent, cu=cu, **hints)
        assert torch.equal(c2, chosen)
        check_attend(st, q, new, o2, chosen=got)


@pytest.mark.parametrize("pages,new", [(700, 3), (4500, 1), (4500, 2), (16000, 1)])
def test_topk_of_long_tables(kv, pages, new):
    """Few pages in the pool, many in the table: scores in LDS or in memory, and many that are equal."""
    D, page, top = 64, 32, 9
    rng = np.random.default_rng(30)
    st = Store(kv, 31, "bf16", 1, D, page, (page * 50,))
    order = rng.integers(0, 50, pages)
    table = st.table[:, torch.from_numpy(order).cuda()].contiguous()
    length = pages * page - 5
    long = Store.__new__(Store)
    long.__dict__.update(st.__dict__, lens=[length])
    rows = (order[:, None] * page + np.arange(page)).reshape(-1)[:length]
    long.k, long.v = [st.k[0][rows]], [st.v[0][rows]]
    q = queries(32, "bf16", (new,), 3, D).cuda()
    out, chosen = st.cache.attend_topk(q, table, i32([length]), top, first=1, recent=2, max_len=length)
    got = chosen.cpu().numpy()
    fifty = st.bounds(0, 0)
    for i in range(new):
        seen = (length - new + i) // page + 1
        want = plain.choose(q[i].double().cpu().numpy(), [fifty[j] for j in order], seen, top, 1, 2)
        assert got[i, 0].tolist() == want
    check_attend(long, q, (new,), out, chosen=got)


def test_topk_by_a_full_lds(kv):
    """Hints decide where scores lie, not what is chosen: a table whose scores fill a workgroup's LDS, and the same by way of memory."""
    D, page, top, pages = 64, 32, 9, 15000
    rng = np.random.default_rng(33)
    st = Store(kv, 34, "bf16", 1, D, page, (page * 50,))
    order = rng.integers(0, 50, pages)
    table = st.table[:, torch.from_numpy(order).cuda()].contiguous()
    length = pages * page - 5
    for new in (1, 2):
        q = queries(35, "bf16", (new,), 3, D).cuda()
        _, chosen = st.cache.attend_topk(q, table, i32([length]), top, max_len=1)
        fifty = st.bounds(0, 0)
        for i in range(new):
            seen = (length - new + i) // page + 1
            assert chosen[i, 0].tolist() == plain.choose(q[i].double().cpu().numpy(), [fifty[j] for j in order], seen, top, 1, 1)
        assert torch.equal(chosen, st.cache.attend_topk(q, table, i32([length]), top)[1])


@pytest.mark.parametrize("dtype,Hq,heads,D,lens,new,top", [
    ("f16", 8, 2, 64, (4000, 3500), (1, 1), 60), ("f32", 4, 2, 128, (2500, 2900, 17), (2, 2, 2), 50), ("bf16", 6, 3, 256, (3000, 2222), (1, 1), 48),
    ("f32", 5, 1, 256, (2600,), (3,), 47), ("bf16", 36, 2, 128, (1900, 2000, 2600), (2, 2, 2), 46), ("f32", 3, 1, 64, (40, 3300), (1, 1), 47)])
def test_few_rows_share_the_card(kv, dtype, Hq, heads, D, lens, new, top):
    """Few rows of many tokens or pages, in equal shares of all tiles; more rows a head than 16 among them."""
    st = Store(kv, 51, dtype, heads, D, 64, lens)
    q = queries(52, dtype, new, Hq, D).cuda()
    lse = torch.empty(q.shape[:2], device="cuda")
    out = st.cache.attend(q, st.table, st.lengths(), lse=lse)
    check_attend(st, q, new, out, lse)
    out, chosen = st.cache.attend_topk(q, st.table, st.lengths(), top, lse=lse)
    check_attend(st, q, new, out, lse, chosen=chosen.cpu().numpy())


def test_topk_ties_take_the_lowest_page(kv):
    """Equal pages score alike: the lowest of them are taken; all-zero queries and keys too."""
    D, page = 64, 32
    c = kv.KvCache(40, 1, D, page)
    x = torch.randn(page, 1, D, device="cuda").repeat(40, 1, 1)
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(1, 2, D, device="cuda")
    for k, qq in ((x, q), (x, q * 0), (x * 0, q)):
        c.append(k, k, table, i32([0]))
        _, chosen = c.attend_topk(qq, table, i32([40 * page]), 5, first=0, recent=1)
        assert chosen.flatten().tolist() == [0, 1, 2, 3, 39]


def test_topk_takes_pages_that_are_not_finite(kv):
    st = Store(kv, 17, "f32", 1, 64, 32, (640,))
    k = torch.randn(1, 1, 64, device="cuda")
    k[0, 0, 3] = float("nan")
    st.cache.append(k, k, st.table, i32([32 * 11 + 31]))
    q = queries(18, "f32", (1,), 2, 64).cuda()
    out, chosen = st.cache.attend_topk(q, st.table, st.lengths(), 4)
    assert 11 in chosen.flatten().tolist() and torch.isnan(out).all()


def test_topk_of_everything_is_attend(kv):
    st = Store(kv, 19, "bf16", 2, 128, 64, (1000, 77))
    q = queries(20, "bf16", (3, 3), 8, 128).cuda()
    out, chosen = st.cache.attend_topk(q, st.table, st.lengths(), 16)
    check_attend(st, q, (3, 3), out)
    check_attend(st, q, (3, 3), st.cache.attend(q, st.table, st.lengths()))


# ---- together ---------------------------------------------------------------------------------
@pytest.mark.parametrize("D,page,dtype", [(128, 64, "bf16"), (64, 32, "f16")])
def test_serving_run(kv, D, page, dtype):
    """Prompts, then tokens one by one: append, attend over everything, attend over chosen pages, at every step."""
    Hq, heads, lens, steps = 8, 2, [90, 1, 200], 40
    st = Store(kv, 21, dtype, heads, D, page, lens, width=8)
    free = iter(range(st.n_pages, st.n_pages + 20))
    big = kv.KvCache(st.n_pages + 20, heads, D, page)
    big.pool.fill_(255)
    big.pool[:st.n_pages], big.bounds[:st.n_pages], big.bound_exps[:st.n_pages] = st.cache.pool, st.cache.bounds, st.cache.bound_exps
    st.cache = big
    rng = np.random.default_rng(22)
    for _ in range(steps):
        for s, n in enumerate(st.lens):
            if n % page == 0:
                st.table[s, n // page] = next(free)
        k, v = (torch.from_numpy(rng.standard_normal((3, heads, D))).to(DT[dtype]) for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((3, Hq, D))).to(DT[dtype]).cuda()
        st.cache.append(k.cuda(), v.cuda(), st.table, st.lengths())
        for s in range(3):
            st.k[s] = np.concatenate([st.k[s], plain.stored(k[s:s + 1].double().numpy())])
            st.v[s] = np.concatenate([st.v[s], plain.stored(v[s:s + 1].double().numpy())])
            st.lens[s] += 1
        check_attend(st, q, (1, 1, 1), st.cache.attend(q, st.table, st.lengths()))
        out, chosen = st.cache.attend_topk(q, st.table, st.lengths(), 2)
        check_attend(st, q, (1, 1, 1), out, chosen=chosen.cpu().numpy())


def test_another_stream(kv):
    st = Store(kv, 23, "bf16", 2, 128, 64, (3000, 500))
    q = queries(24, "bf16", (1, 1), 8, 128).cuda()
    want = st.cache.attend(q, st.table, st.lengths())
    wk, wc = st.cache.attend_topk(q, st.table, st.lengths(), 6)
    lens = st.lengths()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = st.cache.attend(q, st.table, lens)
        gk, gc = st.cache.attend_topk(q, st.table, lens, 6)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(gk, wk) and torch.equal(gc, wc)
    # by handle, while the current stream allocates and writes: no call's scratch is handed to another stream
    other = torch.cuda.Stream()
    outs = []
    for _ in range(20):
        outs.append(st.cache.attend(q, st.table, lens, stream=other.cuda_stream))
        outs.append(st.cache.attend_topk(q, st.table, lens, 6, stream=other.cuda_stream)[0])
        junk = [torch.full((1 << 16,), 7, dtype=torch.uint8, device="cuda") for _ in range(8)]
        del junk
    torch.cuda.synchronize()
    assert all(torch.equal(o, want if i % 2 == 0 else wk) for i, o in enumerate(outs))
    assert torch.equal(st.cache.attend(q, st.table, lens, stream=0), want)


def test_captured_and_replayed(kv):
    """A step in a graph: replayed on new tokens, lengths and queries, beside eager work and a second graph."""
    D, Hq, heads, page = 128, 8, 2, 64
    st = Store(kv, 25, "bf16", heads, D, page, (2000, 130), width=40)
    st.table[0, 32:] = -1
    k, v, q = (torch.zeros(2, h, D, dtype=torch.bfloat16, device="cuda") for h in (heads, heads, Hq))
    before, after = st.lengths(), st.lengths() + 1

    def step():
        st.cache.append(k, v, st.table, before)
        a = st.cache.attend(q, st.table, after)
        b, c = st.cache.attend_topk(q, st.table, after, 5)
        return a, b, c

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for i in range(6):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, device="cuda").to(t.dtype))
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        g, outs = graphs[i % 2]
        for x in outs:
            x.fill_(1)
        g.replay()
        junk = torch.randn(1 << 20, device="cuda").sum()  # eager work between the replays
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(x, y), i
        before += 1
        after += 1
        del junk


def test_python_refusals(kv):
    from gvdb import InvalidArgument

    st = Store(kv, 26, "bf16", 2, 64, 32, (40, 9))
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    c, t, n = st.cache, st.table, st.lengths()
    for bad in (lambda: c.attend(q.double(), t, n), lambda: c.attend(q[:, :3], t, n), lambda: c.attend(q[..., ::2], t, n),
                lambda: c.attend(q.cpu(), t, n), lambda: c.attend(q, t.long(), n), lambda: c.attend(q, t, n[:1]),
                lambda: c.attend(q, t, n, cu=n), lambda: c.attend(q, t, n, out=q.float()), lambda: c.attend(q[:1], t, n),
                lambda: c.attend(q, t, n, lse=torch.zeros(2, 3, device="cuda")), lambda: c.attend_topk(q, t, n, 0),
                lambda: c.attend_topk(q, t, n, 2, first=2, recent=1), lambda: c.append(q[:, :2], q, t, n),
                lambda: c.append(q[:, :2], q[:, :2].float(), t, n), lambda: c.attend(q, t.t(), n),
                lambda: kv.KvCache(4, 2, 96), lambda: kv.KvCache(4, 2, 64, 2048), lambda: kv.KvCache(0, 2, 64), lambda: kv.KvCache(4, 5000, 64),
                lambda: c.attend(q, t, n, out=q[:1].expand(2, 4, 64)), lambda: c.read(t, n, 2, out=(q[:, :1].expand(2, 2, 64), q[:, :2])), lambda: kv.KvCache.from_buffers(c.pool, c.bounds[:1], c.bound_exps)):
        with pytest.raises((InvalidArgument, Exception)) as e:
            bad()
        assert "VectorDbError" in [k.__name__ for k in type(e.value).__mro__], e.value
