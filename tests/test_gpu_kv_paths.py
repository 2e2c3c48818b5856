"""GPU: what every path of the token cache's attention has to keep alike, whatever the launch was sized for."""
import numpy as np
import pytest
import torch

import kv_plain as plain
from test_gpu_kv import DT, HALF, TINY, i32, kv  # noqa: F401  (kv: the fixture)

pytestmark = pytest.mark.gpu


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
