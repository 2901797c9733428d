"""GPU tests of attention over the 4-bit cache at the ends of the format's range: scale
bytes near 0 and 252 in keys and values, and scores of any finite size."""
import math

import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.conv import DType
from tests.mx4_util import DTS, IDS, TORCH, blocks_of, pack
from tests.test_gpu_kv4 import Case, DEV, HEADS, i32

pytestmark = pytest.mark.gpu


def rescale(c, which, byte):
    """All live scales of the keys (0) or values (1) moved alike, so that the largest is `byte`: by that power of two."""
    s = c.cache[2 * which + 1]
    live = s != 255
    by = byte - int(s[live].max())
    s[live] = (s[live].int() + by).to(torch.uint8)
    assert s[live].max() == byte and byte - s[live].min().int() < 20  # nothing wrapped
    return by


@pytest.mark.parametrize("dt", [DType.F32, DType.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d, q_lens, k_lens", [
    (64, [1, 1, 1], [300, 31, 1]), (128, [1, 2], [3000, 700]), (96, [70, 3], [70, 260]), (256, [40, 1], [100, 1500])])
@pytest.mark.parametrize("byte", [252, 245, 200, 60, 30, 20])
def test_values_of_any_size(byte, d, q_lens, k_lens, dt):
    # a mean of values is never larger than they are: up to 6 * 2^125, with as many keys as there may be
    hq, hkv = HEADS[d // 32 % 4]
    c = Case(byte + d, q_lens, k_lens, hq, hkv, d, dt)
    want, tol = c.want()
    by = 2.0 ** rescale(c, 1, byte)  # result and bound are proportional to the values
    got = c.run().double()
    # and what fp32's smallest numbers lose: half of 2^-149 a key, in units of a largest probability of 2^-5 divided by
    # the keys, as a power of two
    n = max(k_lens)
    tol = tol * by + 2.0 ** -150 * n * 2.0 ** (math.ceil(math.log2(max(n, 32))) + 6)
    assert torch.isfinite(got).all()
    over = (got - want * by).abs() / tol
    assert (over <= 1).all(), over.max().item()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_values_that_are_too_small_read_as_zero(dt):
    # 300 keys: below scale bytes of 5 + 9; beside them ordinary values and NaN count as ever
    c = Case(23, [1, 1, 20], [300, 40, 60], 4, 2, 64, dt)
    s = c.cache[3]
    small = (torch.arange(s.shape[0])[:, None, None, None] % 2 == 1) & (s != 255)
    s[small] = 9
    c.cache[3][c.table[0, 3], 1, 4, 1] = 255
    got = c.run().double()
    c.cache[2][(s == 9).repeat_interleave(16, -1)] = 0
    assert (s == 9).any() and torch.isnan(got).any() and not torch.isnan(got).all()
    c.check(got)


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_equal_values_at_the_top_of_the_range(dt):
    # every key alike: the mean of 20000 equal values is that value
    top = 252 if dt != DType.F16 else 127 + 12
    n, d, hkv, page = 20000, 64, 2, 64
    pages = -(-n // page)
    cache = mx4.kv4_cache(pages, page, hkv, d)
    cache[0].fill_(0x22), cache[1].fill_(127), cache[2].fill_(0x77), cache[3].fill_(top)
    q = torch.randn(5, 4, d, generator=torch.Generator().manual_seed(1)).to(TORCH[dt]).to(DEV)
    out = torch.empty_like(q)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(3, 1)
    spec = mx4.Kv4AttnSpec(nseq=3, tokens=5, hq=4, hkv=hkv, d=d, page=page, pages=pages, table_width=pages, dt=dt)
    spec.run(q, *cache, i32([0, 1, 2, 5]), table, i32([n, 1, 333]), out)
    want = 6 * 2.0 ** (top - 127)
    # n probabilities of one size in numerator and denominator: the sums' roundings, a quarter of the keys in a chain
    # of 32s and the parts', and the store's
    tol = 2.0 ** -23 * (n / 32 / 4 + 64) + torch.finfo(TORCH[dt]).eps / 2 + (2.0 ** -15 if dt == DType.F16 else 0)
    assert ((out.double() / want - 1).abs() <= tol).all(), (out.double() / want - 1).abs().max().item()


@pytest.mark.parametrize("dt", [DType.F32, DType.BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("byte, power", [(0, 124), (3, 120), (40, 90), (200, -72), (240, -110)])
def test_keys_of_any_size(byte, power, dt):
    # small keys under large queries and the other way round: the scores are ordinary
    c = Case(byte + 31, [1, 33, 2], [200, 90, 1200], 4, 2, 96, dt)
    s = c.cache[1]
    s[s != 255] = byte
    c.q = (c.q.float() * 2.0 ** power).to(TORCH[dt])
    assert torch.isfinite(c.q).all() and c.q.abs().max() > 0
    c.check()


class Known(Case):
    """Each (row, head) has one key, at `copies` places, that scores highest by half a unit at least, before the scale;
    all products are exact in fp32."""

    def __init__(self, seed, q_lens, k_lens, hq, hkv, d, dt, scale, copies=1, **kw):
        super().__init__(seed, q_lens, k_lens, hq, hkv, d, dt, scale=scale, **kw)
        g = torch.Generator().manual_seed(seed)
        self.q[:, :hq * d] = (torch.randint(0, 2, (self.tokens, hq * d), generator=g) * 2 - 1).to(self.q.dtype)
        codes, scales = self.cache[0], self.cache[1]
        scales[scales != 255] = 127
        # all others' elements are 3 at most
        codes &= 0xdd
        self.best = torch.zeros(self.tokens, hq, copies, dtype=torch.long)
        for b, (lq, lk) in enumerate(zip(q_lens, k_lens)):
            at = torch.randperm(lk - lq + 1, generator=g)[:lq * hq * copies].view(lq, hq, copies)  # keys that all rows see
            for i in range(lq):
                for h in range(hq):
                    j, t = at[i, h], self.q_start[b] + i
                    row = self.q[t, h * d:(h + 1) * d].double() * 6  # the key along the query: 6 d
                    cc, ss = blocks_of(row.view(-1, 32))
                    assert (ss == 127).all()
                    p = self.table[b].long()[j // self.page]
                    codes[p, h // (hq // hkv), j % self.page] = pack(cc).flatten()
                    self.best[t, h] = j

    def best_values(self):
        out = torch.zeros(self.tokens, self.hq, self.d, dtype=torch.float64)
        for b, lq in enumerate(self.q_lens):
            k, v, _ = self.held(b)
            for i in range(lq):
                t = self.q_start[b] + i
                for h in range(self.hq):
                    kh = h // (self.hq // self.hkv)
                    s = k[:, kh] @ self.q[t, h * self.d:(h + 1) * self.d].double()
                    best = self.best[t, h]
                    top = s.topk(len(best) + 1)
                    assert set(top.indices[:-1].tolist()) == set(best.tolist()) and top.values[-2] - top.values[-1] >= 0.5
                    out[t, h] = v[best, kh].mean(0)
        return out


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("q_lens, k_lens", [([3, 1], [200, 333]), ([1], [2500]), ([30, 12], [400, 70])])
@pytest.mark.parametrize("scale", [1e3, 1e4, 1e6, 1e10, 1e18])
def test_large_scores(scale, q_lens, k_lens, dt):
    # the best key leads by 500 or more: the others' probabilities are 0 and the result is its value
    c = Known(41, q_lens, k_lens, 4, 2, 64, dt, scale)
    got, want = c.run().double(), c.best_values()
    # one probability in numerator and denominator: f16 cuts it to 16 bits and sums it whole; a quotient and a store
    tol = 2.0 ** -22 + torch.finfo(TORCH[dt]).eps / 2 + (2.0 ** -15 if dt == DType.F16 else 0)
    assert ((got - want).abs() <= tol * want.abs() + 1e-30).all(), (got - want).abs().max().item()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("scale", [1e2, 777.0, 12345.0, 3e7])
def test_equal_scores_in_other_wavefronts_and_parts(scale, dt):
    # the same best key at five places, some in other wavefronts or parts: the mean of its values
    c = Known(43, [2, 1], [400, 3000], 4, 2, 64, dt, scale, copies=5)
    assert c.spec().plan().parts > 1
    got, want = c.run().double(), c.best_values()
    # the exponential's argument, (score * scale less the maximum), is the same for equal scores wherever they are but
    # for a wavefront's own rounding of the maximum, half a unit of its last place at the most, by which its
    # probabilities and the factor that joins them differ: nothing is left of it. Sums of five, a quotient, a store
    u = {DType.F32: 0.0, DType.F16: 2.0 ** -15, DType.BF16: 2.0 ** -8}[dt]
    mag = torch.stack([v.abs() for v in (want, got)]).amax(0) + 6.0
    assert ((got - want).abs() <= (2 * u + 2.0 ** -20) * mag + torch.finfo(TORCH[dt]).eps / 2 * want.abs()).all()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_scores_of_some_hundreds(dt):
    c = Case(7, [3, 1], [200, 333], 4, 2, 64, dt, scale=3.0)
    got = c.run().double()
    want, tol = c.want()
    if dt == DType.F16:  # results below f16's smallest normal number are stored in steps of 2^-24
        tol = tol + 2.0 ** -25
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("step", [0.05, 0.5, 3.0, 40.0, 1e5])
def test_a_maximum_that_rises_with_every_key(step, dt):
    # key j scores j steps, exactly: its digits to the base of 4 are one element of a block each
    n, d, dig = 900, 160, 5
    c = Case(51, [2, 1, 40], [n, 50, 333], 2, 1, d, dt, scale=step)
    for b, lk in enumerate(c.k_lens):
        j = torch.arange(lk)
        x = torch.zeros(lk, d)
        for i in range(dig):
            x[:, 32 * i] = (j // 4 ** i % 4 * 4 ** i).float()
        cc, ss = blocks_of(x.view(lk, dig, 32))
        at = c.table[b].long()[j // c.page]
        c.cache[0][at, 0, j % c.page], c.cache[1][at, 0, j % c.page] = pack(cc).flatten(-2), ss
    c.q[:] = 0
    for h in range(2):
        c.q[:, h * d:(h + 1) * d:32] = 1 - 2 * h  # the second head's scores fall
    got = c.run().double()
    # the scale's rounding, 2^-24 of an exponent that counts only down to some -60, and the exponential; the sums
    u = {DType.F32: 0.0, DType.F16: 2.0 ** -15, DType.BF16: 2.0 ** -8}[dt]
    rel = 2 * (u + 64 * 2.0 ** -23) + (n / 4 + 64) * 2.0 ** -23
    for b, (lq, lk) in enumerate(zip(c.q_lens, c.k_lens)):
        v = c.held(b)[1][:, 0]
        for h in range(2):
            j = torch.arange(lk)
            s = torch.where(j[None] <= torch.arange(lq)[:, None] + lk - lq, (1 - 2 * h) * j.double()[None] * step, -math.inf)
            p = torch.softmax(s, -1)
            t = c.q_start[b]
            want = p @ v
            tol = rel * (p @ v.abs()) + torch.finfo(TORCH[dt]).eps / 2 * want.abs() + 1e-12
            over = (got[t:t + lq, h] - want).abs() / tol
            assert (over <= 1).all(), (b, h, over.max().item())
