"""GPU: what every path of the token cache's attention has to keep alike, whatever the launch was sized for."""
import ctypes

import numpy as np
import pytest
import torch

import kv_plain as plain
import test_gpu_kv
from test_gpu_kv import DT, HALF, TINY, Store, check_attend, i32, kv, queries  # noqa: F401  (kv: the fixture)

pytestmark = pytest.mark.gpu

UNITS, PARTS, LINE, ROWS, ROW_PARTS = range(5)  # enum gvdb_kv_path


@pytest.fixture(autouse=True)
def sixteen_bits(monkeypatch):
    """What `check_attend` allows for the probabilities' bits: bf16 rows have as many as f16's on every path."""
    monkeypatch.setitem(test_gpu_kv.PROB, "bf16", 2.0 ** -16)


def path(cache, q, table, lens, cu=None, max_new=0, max_len=0, top=0):
    batch, _ = cache._batch(table, lens, cu, q.shape[0], max_new, max_len)
    got = ctypes.c_uint32(99)
    assert cache._lib.gvdb_kv_attend_path(cache._ref, batch, cache._codes[q.dtype], q.shape[1], top, ctypes.byref(got)) == 0
    return got.value


class Cancelling:
    """One sequence of `n` tokens whose values nearly cancel, channel by channel, under one query's probabilities: what is left is at
    most a sixty-fourth of the sum of their magnitudes, so that an output's own rounding hides nothing.  With 8 bits of each
    probability the outputs are 2 to 9 times as far off as `check` allows, with 16 a tenth of it."""

    def __init__(self, kv, seed, dtype, heads, D, page, n, width, scale=None):  # noqa: F811
        rng = np.random.default_rng(seed)
        self.scale = D ** -0.5 if scale is None else scale
        k = torch.from_numpy(rng.standard_normal((n, heads, D))).to(DT[dtype])
        self.k = plain.stored(k.double().numpy())
        self.q = torch.from_numpy(rng.standard_normal((heads, D)) * (1.0 if D == 64 else 0.5)).to(DT[dtype])
        self.v = np.zeros((n, heads, D))
        for h in range(heads):
            p = np.exp((self.k[:, h] @ self.q[h].double().numpy()) * self.scale)
            left = np.zeros(D)
            for j in np.argsort(-p):
                self.v[j, h] = -np.where(left == 0, rng.choice([-1, 1], D), np.sign(left)) * rng.choice([2.0, 3.0, 4.0, 6.0], D)
                left += p[j] * self.v[j, h]
        assert (plain.stored(self.v) == self.v).all()
        need = -(-n // page)
        self.cache = kv.KvCache(need, heads, D, page)
        self.table = torch.full((1, width), -1, dtype=torch.int32)
        self.table[0, :need] = torch.from_numpy(rng.permutation(need).astype(np.int32))
        self.table = self.table.cuda()
        self.cache.append(k.cuda(), torch.from_numpy(self.v).to(DT[dtype]).cuda(), self.table, i32([0]))
        self.n, self.heads, self.D, self.dtype = n, heads, D, dtype

    def rows(self, count, group):
        """[count, heads * group, D]: the one query everywhere."""
        return self.q.repeat_interleave(group, 0)[None].repeat(count, 1, 1).cuda()

    def check(self, out, group):
        out = out.double().cpu().numpy()
        for h in range(self.heads):
            o, _, absum, s1 = plain.attend(self.q[h].double().numpy(), self.k[:, h], self.v[:, h], self.scale, np.ones(self.n, bool))
            assert (np.abs(o) <= 2.0 ** -6 * absum).all()
            # scores and sums in 32 bits as elsewhere; a probability in 16 bits is off by 2^-16 of itself at most
            rel = 2 * (self.D + 8) * 2.0 ** -24 * s1 + (self.n / 32 + 64) * 2.0 ** -23
            bound = HALF[self.dtype] * np.abs(o) + (2.0 ** -16 + rel) * (1 + HALF[self.dtype]) * absum + TINY[self.dtype]
            worst = (np.abs(out[:, h * group:(h + 1) * group] - o) / bound).max()
            assert worst <= 1, (h, float(worst))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D,heads,group,page,n,seqs,rows", [
    (128, 2, 4, 64, 90, 2, 1),       # single tokens
    (64, 1, 8, 32, 150, 40, 1),
    (256, 1, 6, 64, 90, 5, 3),       # a few
    (64, 1, 32, 64, 150, 2, 64),     # prompts: by 128 rows or by 16, as the hints have it
    (128, 1, 8, 64, 90, 96, 128),
    (64, 1, 8, 32, 150, 96, 128),
    (256, 1, 8, 64, 90, 64, 128),
    (128, 1, 16, 32, 90, 2, 40),
])
def test_probabilities_have_16_bits_on_every_path(kv, dtype, D, heads, group, page, n, seqs, rows):  # noqa: F811
    """Neither hints nor the batch decide how many bits a probability has: tables far wider than the sequences, and hints that are right,
    far too small and missing."""
    for width in (-(-n // page), 300):
        st = Cancelling(kv, 60, dtype, heads, D, page, n, width)
        q = st.rows(seqs * rows, group)
        table, lens = st.table.expand(seqs, -1).contiguous(), i32([n] * seqs)
        for cu in (None, i32(np.arange(seqs + 1) * rows)):
            for hints in ({}, {"max_new": rows, "max_len": n}, {"max_new": 1, "max_len": 1}):
                st.check(st.cache.attend(q, table, lens, cu=cu, causal=False, **hints), group)
        if rows == 1:  # every page chosen
            st.check(st.cache.attend_topk(q, table, lens, -(-n // page))[0], group)


# ---- 128 rows a workgroup ---------------------------------------------------------------------
class Crowd:
    """The sequences of a Store `copies` times over, between `before` and `behind` rows of no sequence: enough rows for workgroups of
    128, or (ROW_PARTS) a table far wider than the sequences.  Every copy's outputs are the first's bits, and the first is checked."""

    def __init__(self, kv, want, seed, dtype, Hq, heads, D, page, lens, new, copies, before=0, behind=0):  # noqa: F811
        width = 4000 if want == ROW_PARTS else None
        self.st = Store(kv, seed, dtype, heads, D, page, lens, width=width)
        self.cache, self.dtype, self.new, self.copies, self.want = self.st.cache, dtype, tuple(new), copies, want
        one = queries(seed + 1, dtype, new, Hq, D)
        rest = queries(seed + 2, dtype, (before + behind + 1,), Hq, D)
        self.one, self.rows, self.before, self.behind = one.cuda(), len(one), before, behind
        self.q = torch.cat((rest[:before], one.repeat(copies, 1, 1), rest[before:before + behind])).cuda()
        self.table, self.lens = self.st.table.repeat(copies, 1), self.st.lengths().repeat(copies)
        self.cu = i32((before + np.cumsum((0,) + self.new * copies)).tolist())
        self.hints = {"max_new": max(new)} if want == ROW_PARTS else {"max_new": max(new), "max_len": max(max(lens), 1)}

    def attend(self, q=None, lens=None, table=None, want=None, **more):
        q, lens, table = self.q if q is None else q, self.lens if lens is None else lens, self.table if table is None else table
        more = {**self.hints, **more}
        assert path(self.cache, q, table, lens, self.cu, more["max_new"], more.get("max_len", 0)) == (self.want if want is None else want)
        return self.cache.attend(q, table, lens, cu=self.cu, **more)

    def first(self, x):
        """The first copy's rows of x, after a look at the others."""
        x = x[self.before:self.before + self.copies * self.rows].contiguous()
        bits = x.view(torch.int16 if x.element_size() == 2 else torch.int32).view(self.copies, self.rows, *x.shape[1:])
        assert torch.equal(bits, bits[:1].expand_as(bits))
        return x[:self.rows]

    def check(self, out, lse=None, skip=(), **more):
        check_attend(self.st, self.one, self.new, self.first(out), None if lse is None else self.first(lse), skip=skip, **more)


CROWDS = [  # (path, dtype, query heads, heads, channels, page, lengths, rows, copies): rows before their sequence's first token among them
    (ROWS, "bf16", 16, 1, 64, 32, (150, 30, 0), (64, 40, 64), 32),
    (ROWS, "f16", 8, 2, 128, 64, (400, 9), (128, 70), 32),
    (ROWS, "bf16", 32, 1, 128, 96, (200, 64), (40, 31), 48),
    (ROWS, "f16", 32, 1, 256, 64, (130, 20), (64, 61), 16),
    (ROW_PARTS, "bf16", 32, 1, 64, 64, (600, 20), (40, 33), 1),
    (ROW_PARTS, "f16", 32, 2, 128, 64, (3000, 100), (16, 9), 1),
    (ROW_PARTS, "bf16", 32, 1, 256, 64, (1100, 5), (20, 9), 1),
]


@pytest.mark.parametrize("shape", CROWDS)
def test_rows_strided_misaligned_and_outside(kv, shape):  # noqa: F811
    """Queries inside a fused row and off 16 bytes, outputs inside wider rows, rows of no sequence at both ends: what is beside stays."""
    c = Crowd(kv, shape[0], 70, *shape[1:], before=3, behind=5)
    rows, Hq, D = c.q.shape
    fused = torch.zeros(rows, Hq + 3, D, dtype=c.q.dtype, device="cuda")
    fused[:, 1:Hq + 1] = c.q
    flat = torch.zeros(rows * Hq * D + 1, dtype=c.q.dtype, device="cuda")[1:].view(rows, Hq, D)
    flat.copy_(c.q)
    heads_first = c.q.transpose(0, 1).contiguous().transpose(0, 1)
    outside = [*range(3), *range(rows - 5, rows)]
    for q in (fused[:, 1:Hq + 1], flat, heads_first):
        big = torch.full((rows, Hq, D + 5), 3.0, dtype=q.dtype, device="cuda")
        lse = torch.full((rows, Hq), 3.0, device="cuda")
        c.check(c.attend(q, out=big[:, :, 2:D + 2], lse=lse), lse)
        assert (big[outside] == 3).all() and (big[:, :, :2] == 3).all() and (big[:, :, D + 2:] == 3).all() and (lse[outside] == 3).all()
        lse.fill_(3.0)
        out = c.attend(q, lse=lse)  # the call's own output: rows of no sequence are 0, their logarithm -inf
        c.check(out, lse)
        assert (out[outside] == 0).all() and (lse[outside] == -np.inf).all()


@pytest.mark.parametrize("shape", CROWDS)
def test_rows_with_any_scale_and_mask(kv, shape):  # noqa: F811
    c = Crowd(kv, shape[0], 73, *shape[1:])
    for scale, causal in ((-0.2, True), (-0.05, False), (0.0, True), (0.4, False)):
        lse = torch.empty(c.q.shape[:2], device="cuda")
        c.check(c.attend(scale=scale, causal=causal, lse=lse), lse, scale=scale, causal=causal)


@pytest.mark.parametrize("shape", CROWDS)
def test_rows_write_over_their_queries(kv, shape):  # noqa: F811
    c = Crowd(kv, shape[0], 76, *shape[1:])
    want, own = c.attend(), c.q.clone()
    assert c.attend(own, out=own) is own and torch.equal(own, want)


@pytest.mark.parametrize("shape", CROWDS)
def test_rows_by_any_hint(kv, shape):  # noqa: F811
    """Lengths and rows beyond the hints that the launch was sized for, as a replayed graph has them."""
    c = Crowd(kv, shape[0], 79, *shape[1:])
    seen = set()
    for hints in ({}, {"max_new": 1, "max_len": 1}, {"max_new": 20, "max_len": 64}, {"max_new": 4000000000, "max_len": 4000000000},
                  {"max_new": max(c.new), "max_len": 1}, c.hints):
        lse = torch.empty(c.q.shape[:2], device="cuda")
        c.check(c.cache.attend(c.q, c.table, c.lens, cu=c.cu, lse=lse, **hints), lse)
        seen.add(path(c.cache, c.q, c.table, c.lens, c.cu, **hints))
    assert c.want in seen and len(seen) > 1


@pytest.mark.parametrize("shape", [
    (ROWS, "bf16", 16, 1, 64, 32, (150, 70), (64, 60), 48), (ROWS, "f16", 8, 2, 128, 64, (390, 70), (128, 70), 32),
    (ROWS, "bf16", 32, 1, 256, 64, (130, 40), (64, 60), 16), (ROW_PARTS, "bf16", 32, 1, 64, 128, (150, 40), (64, 33), 1),
    (ROW_PARTS, "f16", 32, 2, 128, 128, (150, 40), (64, 33), 1), (ROW_PARTS, "bf16", 32, 1, 256, 128, (150, 40), (64, 33), 1)])
def test_rows_of_pages_that_are_not_there(kv, shape):  # noqa: F811
    """A page that is not there, and a length that the table does not cover: NaN in the rows that see it, and in no other."""
    c = Crowd(kv, shape[0], 82, *shape[1:])
    S, L, n, page, width = len(c.st.lens), c.st.lens[0], c.new[0], c.st.page, c.table.shape[1]
    for kind in (-1, c.cache.n_pages, "short table"):
        table, lens = c.table.clone(), c.lens.clone()
        if kind == "short table":  # every copy's first sequence ends two tokens behind its table, whose pages are all there
            lens[::S] = width * page + 2
            table[::S, L // page:] = table[0, 0]  # whole, and written
            gone = torch.arange(n) >= n - 2
        else:
            table[::S, 1] = kind
            gone = torch.arange(n) + L - n >= page
        out = c.first(c.attend(lens=lens, table=table))
        assert torch.isnan(out[:n]).flatten(1).all(1).tolist() == gone.tolist(), kind
        assert torch.isfinite(out[:n][~gone]).all()
        check_attend(c.st, c.one, c.new, out, skip={(r, h) for r in range(n) for h in range(c.q.shape[1]) if gone[r] or kind == "short table"})


def test_paths_of_the_other_tests(kv):  # noqa: F811
    """The ways that short calls take: single tokens, few tokens, packed rows, one sequence's prompt in 32 bits."""
    cache = kv.KvCache(8, 8, 128, 64)
    for dtype, seqs, new, width, ragged, max_len, want in (("bf16", 1, 1, 12, False, 768, UNITS), ("bf16", 64, 1, 157, False, 10000, LINE),
                                                            ("f32", 5, 5, 300, True, 19000, PARTS), ("bf16", 2, 2048, 157, False, 10000, ROWS),
                                                            ("f16", 2, 512, 500, True, 32000, ROW_PARTS), ("f32", 2, 2048, 157, False, 10000, UNITS)):
        q = torch.empty(seqs * new, 32, 128, dtype=DT[dtype], device="cuda")
        table, lens = torch.zeros(seqs, width, dtype=torch.int32, device="cuda"), i32([0] * seqs)
        cu = i32((np.arange(seqs + 1) * new).tolist()) if ragged else None
        assert path(cache, q, table, lens, cu, new, max_len) == want, (dtype, seqs, new)


@pytest.mark.parametrize("dtype,Hq,heads,D,new,outside", [("bf16", 3, 1, 64, (700, 1, 1, 600), (2, 3)), ("f16", 20, 1, 128, (1101,), (0, 0)),
                                                           ("f32", 4, 4, 64, (1,) * 300, (0, 4)), ("bf16", 8, 2, 256, (250, 0, 299), (1, 0))])
def test_topk_of_long_tables_in_groups_of_rows(kv, dtype, Hq, heads, D, new, outside):  # noqa: F811
    """More rows than scratch holds the page scores of: groups that end inside a sequence, and inside a workgroup's rows."""
    page, top, fifty, pages = 32, 6, 50, 16100
    rng = np.random.default_rng(90)
    st = Store(kv, 91, dtype, heads, D, page, (page * fifty,))
    order = rng.integers(0, fifty, (len(new), pages))
    table = st.table[0, torch.from_numpy(order).cuda()].contiguous()
    lens = [int(x) for x in rng.integers(pages * page - 200 * page, pages * page, len(new))]
    q = queries(92, dtype, (sum(outside) + sum(new),), Hq, D).cuda()
    cu = i32((outside[0] + np.cumsum((0,) + new)).tolist())
    assert q.shape[0] * heads * pages * 4 > 64 << 20
    out, chosen = st.cache.attend_topk(q, table, i32(lens), top, first=1, recent=1, cu=cu)
    got, qd, g = chosen.cpu().numpy(), q.double().cpu().numpy(), Hq // heads
    bounds = [st.bounds(0, h) for h in range(heads)]
    row = outside[0]
    assert (got[:row] == -1).all() and (out[:row] == 0).all()
    for s, n in enumerate(new):
        for i in range(n):
            limit = lens[s] - n + i + 1
            seen = -(-limit // page)
            for h in range(heads):
                # every page scores as the one of the fifty that it is
                each = scores_of(qd[row, h * g:(h + 1) * g], bounds[h])[order[s, :seen]]
                each[0] = each[seen - 1] = np.inf
                assert got[row, h].tolist() == sorted(np.argsort(-each, kind="stable")[:top].tolist()), (s, i, h)
                if i in (0, n // 2, n - 1) and s < 4:
                    tokens = (got[row, h][:, None] * page + np.arange(page)).reshape(-1)
                    tokens = tokens[tokens < limit]
                    place = order[s][tokens // page] * page + tokens % page
                    for hq in range(h * g, (h + 1) * g):
                        o, _, absum, s1 = plain.attend(qd[row, hq], st.k[0][place][:, h], st.v[0][place][:, h], D ** -0.5, np.ones(len(place), bool))
                        rel = 2 * (D + 8) * 2.0 ** -24 * s1 + (top * page / 32 + 64) * 2.0 ** -23
                        tol = HALF[dtype] * np.abs(o) + (test_gpu_kv.PROB[dtype] + rel) * (1 + HALF[dtype]) * absum + TINY[dtype]
                        assert (np.abs(out[row, hq].double().cpu().numpy() - o) <= tol).all(), (s, i, hq)
            row += 1
    assert (got[row:] == -1).all() and (out[row:] == 0).all()


def scores_of(q, page_bounds):
    """kv_plain.choose's scores of pages whose bounds are finite."""
    score = np.full(len(page_bounds), -np.inf)
    hi, lo = (np.stack([b8[x] for b8, _ in page_bounds]).astype(np.float64) for x in (0, 1))
    unit = 2.0 ** (np.array([e for _, e in page_bounds], np.float64) - 133)
    for row in q:
        a = float(plain.power(np.abs(row).max()))
        q8 = np.rint(row / 2.0 ** a)
        score = np.maximum(score, (hi @ np.maximum(q8, 0) + lo @ np.minimum(q8, 0)) * 2.0 ** a * unit)
    return score


# ---- streams ----------------------------------------------------------------------------------
def test_tensors_dropped_after_a_call_on_another_stream(kv):  # noqa: F811
    """The given stream has other work first; what the call was given is dropped and its size asked for again before it runs."""
    st = Store(kv, 95, "bf16", 2, 128, 64, (3000, 500))
    q, lens = queries(96, "bf16", (1, 1), 8, 128).cuda(), st.lengths()
    want, (wk, wc) = st.cache.attend(q, st.table, lens), st.cache.attend_topk(q, st.table, lens, 6)
    side = torch.cuda.Stream()
    for _ in range(3):
        given = [q.clone(), st.table.clone(), lens.clone()]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        got = st.cache.attend(*given, stream=side.cuda_stream)
        gk, gc = st.cache.attend_topk(*given, 6, stream=side.cuda_stream)
        del given
        junk = [torch.ones_like(x) for x in (q, st.table, lens) for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(gk, wk) and torch.equal(gc, wc)
        del junk


def test_captured_on_a_given_stream(kv):  # noqa: F811
    st = Store(kv, 97, "bf16", 2, 128, 64, (3000, 500))
    q, lens = queries(98, "bf16", (1, 1), 8, 128).cuda(), st.lengths()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    st.cache.attend(q, st.table, lens, stream=side.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = st.cache.attend(q, st.table, lens, stream=side.cuda_stream)
        pages = st.cache.attend_topk(q, st.table, lens, 6, stream=side.cuda_stream)
    for i in range(4):
        q.copy_(queries(99 + i, "bf16", (1, 1), 8, 128))
        want, (wk, wc) = st.cache.attend(q, st.table, lens), st.cache.attend_topk(q, st.table, lens, 6)
        out.fill_(1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pages[0], wk) and torch.equal(pages[1], wc), i


# ---- append, read: the ends of the 16-bit types -----------------------------------------------
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_append_of_subnormal_and_extreme_16_bit_values(kv, dtype, D):  # noqa: F811
    """Every bit pattern of the type in groups of its own size and beside larger and smaller ones, infinities and NaN among them."""
    rng = np.random.default_rng(110)
    bits = np.arange(1 << 16, dtype=np.uint32).astype(np.uint16)
    width = 10 if dtype == "f16" else 7
    exps = (bits >> width) & ((1 << (15 - width)) - 1)
    groups = [rng.permutation(bits[exps == e])[:2048].reshape(-1, 32) for e in range(exps.max() + 1) if (exps == e).sum() >= 32]
    small = bits[exps <= 1]
    groups += [rng.choice(small, (400, 32)), rng.choice(bits[exps < exps.max()], (400, 32))]
    mixed = rng.choice(small, (60, 32))
    mixed[:, 5] = rng.choice(bits[(exps > 1) & (exps < 12)], 60)
    few = np.zeros((40, 32), np.uint16)  # almost nothing: a group's only value is one of the smallest
    few[:, 9] = np.r_[np.arange(1, 31), 0x8000 + np.arange(1, 11)]
    x = np.concatenate(groups + [mixed, few])
    x = x[:len(x) // (D // 32) * (D // 32)].reshape(-1, 1, D)
    t = torch.from_numpy(x.view(np.int16)).view(DT[dtype])
    n, page = len(x), 64
    need = -(-n // page)
    cache, table = kv.KvCache(need, 1, D, page), torch.arange(need, dtype=torch.int32, device="cuda")[None]
    cache.append(t.cuda(), t.flip(0).cuda(), table, i32([0]))
    k, v = cache.read(table, i32([0]), n, dtype=torch.float32)
    want = plain.stored(t.double().numpy())
    assert np.array_equal(k.double().cpu().numpy(), want, equal_nan=True)
    assert np.array_equal(v.flip(0).double().cpu().numpy(), want, equal_nan=True)
    assert np.isnan(want).any() and (np.abs(want[np.isfinite(want)]) > 0).any()
    b8, be = cache.bounds.cpu().numpy(), cache.bound_exps.cpu().numpy()
    for j in range(need):
        rows = want[j * page:(j + 1) * page, 0]
        b, e = plain.bounds(rows)
        e = 7 if not rows.any() else e  # nothing but zeros: the smallest power that there is (frexp(0) says 2^0)
        assert be[j, 0] == e and np.array_equal(b8[j, 0], b), j
    # read back in any type: rounded once
    for other in DT.values():
        k, _ = cache.read(table, i32([0]), n, dtype=other)
        finite = torch.from_numpy(want).float()  # exact: a code has two bits, its power of two is 2^-125 at least
        assert torch.equal(k.cpu().nan_to_num(7.0, posinf=8.0, neginf=-8.0), finite.to(other).nan_to_num(7.0, posinf=8.0, neginf=-8.0))


@pytest.mark.parametrize("dtype,Hq,D,new,n", [("f32", 2, 64, 3, 90), ("bf16", 2, 128, 1, 90), ("bf16", 8, 64, 128, 150), ("f32", 1, 256, 1, 3000)])
def test_a_scale_of_nothing_weighs_all_alike(kv, dtype, Hq, D, new, n):  # noqa: F811
    """Whatever the scores are that it is multiplied with; and a scale that is next to nothing is what it is."""
    copies = 96 if new == 128 else 1
    st = Store(kv, 120, dtype, 1, D, 64, (n,))
    big = torch.randn(n, 1, D, generator=torch.Generator().manual_seed(1)) * 1e17
    big = big.to(DT[dtype])
    v = torch.randn(n, 1, D, generator=torch.Generator().manual_seed(2)).to(DT[dtype])
    st.cache.append(big.cuda(), v.cuda(), st.table, i32([0]))
    st.k[0], st.v[0] = plain.stored(big.double().numpy()), plain.stored(v.double().numpy())
    q = (queries(121, dtype, (new,), Hq, D).float() * 1e18).to(DT[dtype])
    table, lens = st.table.repeat(copies, 1), i32([n] * copies)
    for scale in (0.0, -0.0, 1e-40, 3e-37):
        out = st.cache.attend(q.repeat(copies, 1, 1).cuda(), table, lens, causal=False, scale=scale)
        assert new != 128 or path(st.cache, q.repeat(copies, 1, 1), table, lens) == ROWS
        check_attend(st, q[:4], (min(new, 4),), out[:4], causal=False, scale=float(np.float32(scale)))


@pytest.mark.parametrize("pages,new,max_len", [(60, 1, 0), (60, 9, 0), (700, 1, 0)])
def test_topk_takes_what_is_not_finite_before_scores_that_overflow(kv, pages, new, max_len):  # noqa: F811
    """Scores beyond the range of 32 bits are equal, and less than a page that holds what is not finite, or is not there."""
    D, page = 64, 32
    cache = kv.KvCache(pages, 1, D, page)
    k = torch.full((pages * page, 1, D), 1e14, device="cuda")
    k[(pages - 8) * page + 3, 0, 7] = float("nan")
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    cache.append(k, k, table, i32([0]))
    table[0, pages - 5] = -1
    q = torch.full((new, 2, D), 1e30, device="cuda")
    _, chosen = cache.attend_topk(q, table, i32([pages * page]), 6, first=0, recent=1, max_len=max_len)
    assert chosen[:, 0].tolist() == [[0, 1, 2, pages - 8, pages - 5, pages - 1]] * new


# ---- calls that are allowed and rarely made ---------------------------------------------------
@pytest.mark.parametrize("dtype,Hq,heads,D,page", [("bf16", 32, 1, 64, 64), ("f16", 32, 2, 128, 32), ("bf16", 32, 1, 256, 64)])
def test_what_is_masked_in_parts_of_rows_may_hold_anything(kv, dtype, Hq, heads, D, page):  # noqa: F811
    for poison in (float("nan"), float("inf"), -float("inf")):
        c = Crowd(kv, ROW_PARTS, 130, dtype, Hq, heads, D, page, (150, 40), (80, 9), 1)
        st = c.st
        k = torch.from_numpy(np.random.default_rng(1).standard_normal((4, heads, D))).to(DT[dtype]).cuda()
        v = k.clone()
        v[1, :, 40] = poison   # token 121: a value, channels 32 .. 63
        k[3, :, 7] = poison    # token 123: a key
        st.cache.append(k, v, st.table[:1], i32([120]))
        st.k[0][120:124], st.v[0][120:124] = plain.stored(k.double().cpu().numpy()), plain.stored(v.double().cpu().numpy())
        c.q[5, 1, 0] = poison
        lse = torch.empty(c.q.shape[:2], device="cuda")
        out = c.attend(lse=lse)
        want = np.zeros((89, Hq, D), bool)
        want[51:80, :, 32:64] = True    # row i of the 80 is token 70 + i
        want[53:80] = True
        want[5, 1] = True
        assert np.array_equal(torch.isnan(out).cpu().numpy(), want)
        c.one = c.q
        c.check(out, lse, skip={(r, h) for r in range(51, 80) for h in range(Hq)} | {(5, 1)})


def test_calls_without_rows(kv):  # noqa: F811
    st = Store(kv, 131, "bf16", 2, 64, 32, (40, 9))
    before = [x.clone() for x in (st.cache.pool, st.cache.bounds, st.cache.bound_exps)]
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    for table, lens, cu in ((st.table, st.lengths(), None), (st.table, st.lengths(), i32([0, 0, 0])), (st.table[:0], i32([]), None)):
        st.cache.append(q[:, :2], q[:, :2], table, lens, cu=cu)
        assert st.cache.attend(q, table, lens, cu=cu).shape == (0, 4, 64)
        out, chosen = st.cache.attend_topk(q, table, lens, 3, cu=cu)
        assert out.shape == (0, 4, 64) and chosen.shape == (0, 2, 3)
        assert all(x.shape == (0, 2, 64) for x in st.cache.read(table, lens, 0, cu=cu))
    assert all(torch.equal(a, b) for a, b in zip(before, (st.cache.pool, st.cache.bounds, st.cache.bound_exps)))


@pytest.mark.parametrize("Hq,heads,D,dtype", [(2048, 1, 64, "bf16"), (333, 1, 256, "f32"), (300, 300, 64, "f16")])
def test_many_heads(kv, Hq, heads, D, dtype):  # noqa: F811
    st = Store(kv, 132, dtype, heads, D, 32, (200, 70))
    q, cu = queries(133, dtype, (2, 1), Hq, D).cuda(), i32([0, 2, 3])
    lse = torch.empty(3, Hq, device="cuda")
    skip = {(i, h) for i in range(3) for h in range(Hq) if h % 37}
    check_attend(st, q, (2, 1), st.cache.attend(q, st.table, st.lengths(), cu=cu, lse=lse), lse, skip=skip)
    out, chosen = st.cache.attend_topk(q, st.table, st.lengths(), 3, cu=cu, lse=lse)
    check_attend(st, q, (2, 1), out, lse, chosen=chosen.cpu().numpy(), skip=skip)


def test_row_bounds_and_lengths_that_make_no_sense(kv):  # noqa: F811
    """They lead nowhere outside the tensors, the table and the pool; what they leave in the cache is not checked."""
    for bad in ([0, 3, 1], [-5, 100, 2], [3, 2, 1], [2 ** 31 - 1, 0, 5], [5, -2 ** 31, 5]):
        st = Store(kv, 134, "bf16", 2, 64, 32, (40, 9))
        q, cu = queries(135, "bf16", (5,), 4, 64).cuda(), i32(bad)
        guard = torch.full((7, 4, 64), 3.0, dtype=q.dtype, device="cuda")
        st.cache.attend(q, st.table, st.lengths(), cu=cu, out=guard[1:6])
        st.cache.attend_topk(q, st.table, st.lengths(), 2, cu=cu, out=guard[1:6])
        st.cache.read(st.table, st.zeros(), 5, cu=cu)
        st.cache.append(q[:, :2], q[:, :2], st.table, st.zeros(), cu=cu)
        torch.cuda.synchronize()
        assert (guard[0] == 3).all() and (guard[6] == 3).all()
    for lens, nan in (((-5, 2 ** 31 - 1), [False, True]), ((-2 ** 31, 0), [False, False])):
        st = Store(kv, 136, "bf16", 2, 64, 32, (40, 9))
        q, k = queries(137, "bf16", (2,), 4, 64).cuda(), st.cache.pool.clone()
        for out in (st.cache.attend(q, st.table, i32(lens)), st.cache.attend_topk(q, st.table, i32(lens), 2)[0]):
            assert [bool(torch.isnan(x).all()) for x in out] == nan and bool((out[0] == 0).all())
        st.cache.append(q[:, :2], q[:, :2], st.table[:, :1].contiguous(), i32([2 ** 31 - 1, 33]))  # behind the table: skipped
        assert torch.equal(k, st.cache.pool)


def test_two_threads_at_once(kv):  # noqa: F811
    """Two callers of one cache, each on a stream of its own, with calls that need scratch: neither sees the other's."""
    import threading

    st = Store(kv, 140, "bf16", 2, 128, 64, (3000, 500))
    shapes = [queries(141 + i, "bf16", (1, 1), 8, 128).cuda() for i in range(2)]
    lens = st.lengths()
    want = [(st.cache.attend(q, st.table, lens), *st.cache.attend_topk(q, st.table, lens, 6)) for q in shapes]
    assert path(st.cache, shapes[0], st.table, lens) == LINE
    torch.cuda.synchronize()
    wrong, done = [], []

    def caller(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(60):
                got = (st.cache.attend(shapes[i], st.table, lens), *st.cache.attend_topk(shapes[i], st.table, lens, 6))
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)
        torch.cuda.current_stream().synchronize()
        done.append(i)

    threads = [threading.Thread(target=caller, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert sorted(done) == [0, 1] and not wrong
