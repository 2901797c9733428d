"""GPU tests of the 4-bit paged cache: what appending stores, exactly, and attention
over it against the formula in 64 bits."""
import math
import random

import pytest
import torch

from ai_engine_amd import mx4
from ai_engine_amd.attn_block import rotation_tables
from ai_engine_amd.conv import AihError, DType
from tests.mx4_util import DTS, GRID, IDS, TORCH, blocks_of, pack, values

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- appending

def noise_cache(seed, pages, page, hkv, d):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (pages, hkv, page, n), generator=g, dtype=torch.uint8).to(DEV) for n in (d // 2, d // 32) * 2]


def rotated(y, cos, sin, rot, pairs):
    """y [tokens, heads, d] fp32, the angles' rows per token: every product and sum rounded by itself."""
    if rot == 0:
        return y.clone()
    c, s = cos[:, None], sin[:, None]
    out = y.clone()
    if pairs:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        out[..., 0:rot:2], out[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        a, b = y[..., :rot // 2], y[..., rot // 2:rot]
        out[..., :rot // 2], out[..., rot // 2:rot] = a * c - b * s, a * s + b * c
    return out


def put(cache, which, slots, new, page):
    """The rows `new` [tokens, hkv, d] quantised into a host copy of the cache, dropped where there is no such row."""
    codes, scales = cache[2 * which].cpu().clone(), cache[2 * which + 1].cpu().clone()
    c, s = blocks_of(new.reshape(new.shape[0], new.shape[1], -1, 32))
    c = pack(c).flatten(-2)
    for t, slot in enumerate(slots):
        if 0 <= slot < codes.shape[0] * page:
            codes[slot // page, :, slot % page], scales[slot // page, :, slot % page] = c[t], s[t]
    return codes, scales


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("tokens, hq, hkv, d, rot, pairs, page, pages", [
    (1, 1, 1, 32, 32, False, 16, 1), (7, 4, 2, 64, 64, True, 16, 3), (33, 3, 3, 96, 48, False, 64, 2),
    (8, 32, 8, 128, 128, False, 64, 4), (20, 2, 1, 160, 0, False, 32, 2), (9, 6, 2, 192, 96, True, 16, 9),
    (5, 0, 2, 224, 224, False, 16, 4), (130, 8, 1, 256, 128, False, 256, 1), (50, 5, 5, 32, 16, True, 4096, 1)])
def test_append(tokens, hq, hkv, d, rot, pairs, page, pages, dt):
    g = torch.Generator().manual_seed(tokens + d)
    pad = 8 if (tokens + hkv) % 2 else 0
    x = (torch.randn(tokens, (hq + 2 * hkv) * d + pad, generator=g) * 2).to(TORCH[dt])
    cos, sin = rotation_tables(11, max(rot, 2), device="cpu")
    pos = torch.randint(-2, 14, (tokens,), generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * page + 6, generator=g)[:tokens].int() - 3  # some before, some behind the cache
    assert len(set(slots.tolist())) == tokens
    cache = noise_cache(1, pages, page, hkv, d)
    heads = x[:, :(hq + 2 * hkv) * d].float().view(tokens, -1, d)
    at = pos.clamp(0, 10).long()
    turned = rotated(heads[:, :hq + hkv], cos[at], sin[at], rot, pairs)
    want_k = put(cache, 0, slots.tolist(), turned[:, hq:], page)
    want_v = put(cache, 1, slots.tolist(), heads[:, hq + hkv:], page)
    q = torch.full((tokens + 1, max(hq, 1) * d), 3.0, dtype=TORCH[dt], device=DEV)
    mx4.Kv4AppendSpec(tokens=tokens, hq=hq, hkv=hkv, d=d, page=page, pages=pages, rot=rot, pairs=pairs, dt=dt,
                      positions=11, x_stride=x.shape[1]).run(
        x.to(DEV), None, None, cos.to(DEV), sin.to(DEV), pos.to(DEV), slots.to(DEV), q if hq else None, *cache)
    for got, want in zip(cache, (*want_k, *want_v)):
        assert torch.equal(got.cpu(), want)
    if hq:
        assert torch.equal(q[:tokens].cpu().view(tokens, hq, d), turned[:, :hq].to(TORCH[dt]))
    assert (q[tokens:] == 3).all()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("d, rot, pairs", [(32, 32, False), (64, 32, True), (96, 96, False), (128, 0, False), (256, 256, True)])
def test_append_with_head_norms(d, rot, pairs, dt):
    tokens, hq, hkv, page, pages = 21, 3, 2, 16, 2
    g = torch.Generator().manual_seed(d)
    x = torch.randn(tokens, hq + 2 * hkv, d, generator=g)
    x[3] *= 1e-18 if dt != DType.F16 else 1e-4
    x[4] *= 1e18 if dt != DType.F16 else 1e3
    x = x.to(TORCH[dt])
    wq, wk = ((1 + 0.2 * torch.randn(d, generator=g)).to(TORCH[dt]) for _ in range(2))
    cos, sin = rotation_tables(64, max(rot, 2), device="cpu")
    slots = torch.randperm(pages * page, generator=g)[:tokens].int()
    cache = noise_cache(1, pages, page, hkv, d)
    want_v = put(cache, 1, slots.tolist(), x[:, hq + hkv:].float(), page)
    q = torch.empty(tokens, hq, d, dtype=TORCH[dt], device=DEV)
    eps = 1e-30 if dt != DType.F16 else 1e-6
    mx4.Kv4AppendSpec(tokens=tokens, hq=hq, hkv=hkv, d=d, page=page, pages=pages, rot=rot, pairs=pairs, norm=True, dt=dt,
                      eps=eps, positions=64).run(
        x.to(DEV), wq.to(DEV), wk.to(DEV), cos.to(DEV), sin.to(DEV), None, slots.to(DEV), q, *cache)
    assert torch.equal(cache[2].cpu(), want_v[0]) and torch.equal(cache[3].cpu(), want_v[1])
    y = x[:, :hq + hkv].double()
    w = torch.cat([wq.double().expand(hq, d), wk.double().expand(hkv, d)])
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w
    y = rotated(y, cos[:tokens].double(), sin[:tokens].double(), rot, pairs)
    # fp32 arithmetic: the sum of d squares, the root, three products, two of which are added: (d + 12) 2^-24 of the
    # two numbers' magnitudes at most
    size = y.abs()
    if rot:
        other = y.clone()
        i = torch.arange(rot)
        other[..., :rot] = y[..., i ^ 1] if pairs else y[..., (i + rot // 2) % rot]
        size = size + other.abs()
    err = (d + 12) * 2.0 ** -24 * (2 * size)
    got = q.double().cpu()
    assert ((got - y[:, :hq]).abs() <= err[:, :hq] + torch.finfo(TORCH[dt]).eps / 2 * y[:, :hq].abs() * 1.01 + 1e-38).all()
    # keys: a scale that the error allows, and a value no further off than the nearest one, but for the error
    k, ke = y[:, hq:], err[:, hq:]
    at = slots.long()
    codes = cache[0].cpu()[at // page, :, at % page].reshape(tokens * hkv, d // 2)
    scales = cache[1].cpu()[at // page, :, at % page].reshape(tokens * hkv, d // 32)
    top = k.reshape(-1, d // 32, 32).abs().amax(-1)
    slack = ke.reshape(-1, d // 32, 32).amax(-1)
    lo, hi = (torch.frexp((top + f * slack).clamp(min=0))[1] - 3 + 127 for f in (-1, 1))
    assert ((scales >= lo) & (scales <= hi)).all()
    size = torch.ldexp(torch.ones(scales.shape, dtype=torch.float64), scales.int() - 127).repeat_interleave(32, -1)
    off = (values(codes, scales) - k.reshape(-1, d)).abs()
    a = (k.reshape(-1, d) / size).abs()
    near = ((a[..., None] - GRID).abs().amin(-1) + 1e-12) * size
    assert (off <= near + 2 * ke.reshape(-1, d)).all()


def test_append_nan_and_infinite_heads():
    x = torch.randn(4, 3, 64)
    x[0, 1, 40], x[1, 2, 3], x[2, 1, 0] = float("nan"), float("inf"), float("-inf")
    cache = noise_cache(2, 1, 16, 1, 64)
    want = *put(cache, 0, range(4), x[:, 1:2], 16), *put(cache, 1, range(4), x[:, 2:], 16)
    q = torch.empty(4, 1, 64, device=DEV)
    mx4.Kv4AppendSpec(tokens=4, hq=1, hkv=1, d=64, page=16, pages=1).run(
        x.to(DEV), None, None, None, None, None, i32([0, 1, 2, 3]), q, *cache)
    for got, w in zip(cache, want):
        assert torch.equal(got.cpu(), w)
    assert torch.equal(q.cpu()[:, 0], x[:, 0])


@pytest.mark.parametrize("pairs", [False, True])
def test_append_rotates_queries_in_place(pairs):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(300, 6, 64, generator=g).to(DEV)
    cos, sin = rotation_tables(300, 64, device=DEV)
    spec = dict(tokens=300, hq=2, hkv=2, d=64, rot=64, pairs=pairs, positions=300, page=64, pages=8)
    slots = torch.arange(300, dtype=torch.int32, device=DEV)
    caches = [mx4.kv4_cache(8, 64, 2, 64) for _ in range(2)]
    q = torch.empty(300, 2, 64, device=DEV)
    mx4.Kv4AppendSpec(**spec).run(x, None, None, cos, sin, None, slots, q, *caches[0])
    keep = x.clone()
    mx4.Kv4AppendSpec(**spec, q_stride=6 * 64).run(x, None, None, cos, sin, None, slots, x, *caches[1])
    assert torch.equal(x[:, :2], q) and torch.equal(x[:, 2:], keep[:, 2:])
    assert all(torch.equal(a, b) for a, b in zip(*caches))


# ---------------------------------------------------------------- attention

class Case:
    """Sequences over a cache of random pages; whatever no sequence holds is NaN."""

    def __init__(self, seed, q_lens, k_lens, hq, hkv, d, dt, page=16, causal=True, scale=None, extra=3, pad=0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.k_lens, self.hq, self.hkv, self.d, self.dt = q_lens, k_lens, hq, hkv, d, dt
        self.page, self.causal, self.scale = page, causal, scale or 1 / math.sqrt(d)
        need = [-(-n // page) for n in k_lens]
        self.pages, self.width = sum(need) + extra, max(need + [1]) + 1
        order = list(range(self.pages))
        random.Random(seed).shuffle(order)
        table = torch.randint(-5, self.pages + 5, (len(k_lens), self.width), generator=g, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.table = table
        self.cache = []
        for _ in range(2):
            v = torch.randn(self.pages, hkv, page, d // 32, 32, generator=g)
            c, s = blocks_of(v)
            live = torch.zeros(self.pages, page, dtype=torch.bool)
            for b, n in enumerate(k_lens):
                for j in range(need[b]):
                    live[table[b, j], :min(page, n - j * page)] = True
            s[~live[:, None].expand(-1, hkv, -1)] = 255
            self.cache += [pack(c).flatten(-2).contiguous(), s.contiguous()]
        self.q_start = [0]
        for n in q_lens:
            self.q_start.append(self.q_start[-1] + n)
        self.tokens = self.q_start[-1]
        self.qw = hq * d + pad
        self.q = torch.randn(self.tokens, self.qw, generator=g).to(TORCH[dt])

    def spec(self, **kw):
        return mx4.Kv4AttnSpec(**{**dict(
            nseq=len(self.q_lens), tokens=self.tokens, hq=self.hq, hkv=self.hkv, d=self.d, page=self.page, pages=self.pages,
            table_width=self.width, causal=self.causal, scale=self.scale, dt=self.dt, q_stride=self.qw, o_stride=self.qw,
            max_len=max(self.k_lens + [1])), **kw})

    def run(self, spec=None, stream=None):
        spec = spec or self.spec()
        out = torch.full((self.tokens + 1, self.qw), -9.0, dtype=TORCH[self.dt], device=DEV)
        spec.run(self.q.to(DEV), *(c.to(DEV) for c in self.cache), i32(self.q_start), self.table.to(DEV), i32(self.k_lens), out)
        torch.cuda.synchronize()
        n = self.hq * self.d
        assert (out[self.tokens:] == -9).all() and (out[:, n:] == -9).all()
        return out[:self.tokens, :n].cpu().view(self.tokens, self.hq, self.d)

    def held(self, b):
        """Keys and values of sequence b: [len, hkv, d] fp64, and which of them are there."""
        n = self.k_lens[b]
        j = torch.arange(n)
        p = self.table[b].long()[j // self.page]
        there = (p >= 0) & (p < self.pages)
        out = []
        for w in range(2):
            c = self.cache[2 * w][p.clamp(0, self.pages - 1), :, j % self.page].reshape(n * self.hkv, -1)
            s = self.cache[2 * w + 1][p.clamp(0, self.pages - 1), :, j % self.page].reshape(n * self.hkv, -1)
            out.append(values(c, s).view(n, self.hkv, self.d))
        return *out, there

    def want(self):
        """(output, error allowed) in fp64.

        Scores: a chain of d products in fp32 and the exponent's rounding, (d + 16) 2^-23 of the magnitudes' sum, as an
        absolute error of the exponent and so a relative one of p, in numerator and denominator. A probability is held
        to u: bf16 half a step, f16 two truncated terms (16 bits: 2^-15), fp32 exactly. The sums: a wavefront adds up
        a quarter of the keys, some joins. One rounding at the end."""
        out = torch.zeros(self.tokens, self.hq, self.d, dtype=torch.float64)
        tol = torch.zeros_like(out)
        u = {DType.F32: 0.0, DType.F16: 2.0 ** -15, DType.BF16: 2.0 ** -8}[self.dt]
        for b, (lq, lk) in enumerate(zip(self.q_lens, self.k_lens)):
            if lq == 0 or lk == 0:
                continue
            k, v, there = self.held(b)
            seen = there[None].expand(lq, lk)
            if self.causal:
                seen = seen & (torch.arange(lk)[None] <= torch.arange(lq)[:, None] + lk - lq)
            q0 = self.q_start[b]
            q = self.q[q0:q0 + lq, :self.hq * self.d].double().view(lq, self.hq, self.d)
            for h in range(self.hq):
                kh, vh = k[:, h // (self.hq // self.hkv)], v[:, h // (self.hq // self.hkv)]
                s = q[:, h] @ kh.nan_to_num().t() * self.scale
                s = torch.where(seen, s + 0 * kh.sum(-1), -math.inf)
                top = s.amax(-1, keepdim=True)
                p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                z = p.sum(-1, keepdim=True)
                p = p / torch.where(z == 0, 1.0, z)
                mag = (torch.where(seen, q[:, h].abs() @ kh.nan_to_num().abs().t() * self.scale, 0.0)).amax(-1, keepdim=True)
                ds = (self.d + 16) * 2.0 ** -23 * mag
                pv = torch.where(p[..., None] > 0, p[..., None] * vh.nan_to_num()[None], 0.0).sum(1) if lk <= 64 else p.nan_to_num() @ vh.nan_to_num()
                bad = (seen.double() @ torch.isnan(vh).double()) > 0
                o = torch.where(bad | torch.isnan(p).any(-1, keepdim=True), math.nan, pv)
                a = p.nan_to_num() @ vh.nan_to_num().abs()
                out[q0:q0 + lq, h] = o
                tol[q0:q0 + lq, h] = (2 * u + 2 * ds + (lk / 4 + 64) * 2.0 ** -23) * a + torch.finfo(TORCH[self.dt]).eps / 2 * pv.abs() + 1e-12
        return out, tol

    def check(self, got=None, spec=None):
        got = (self.run(spec) if got is None else got).double()
        want, tol = self.want()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        over = ((got - want).abs() / tol).nan_to_num()
        assert (over <= 1).all(), over.max().item()


HEADS = [(1, 1), (4, 1), (8, 2), (6, 3), (32, 8)]


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 160, 192, 224, 256])
def test_single_tokens(d, dt):
    hq, hkv = HEADS[d // 32 % 5]
    Case(d, [1] * 7, [0, 1, 2, 31, 33, 130, 300], hq, hkv, d, dt, page=16 if d % 64 else 32).check()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_prompts(d, causal, dt):
    hq, hkv = HEADS[d // 32 % 4]
    Case(d + 1, [1, 0, 5, 40, 3, 70], [64, 5, 5, 40, 1, 260], hq, hkv, d, dt, page=16, causal=causal, pad=8).check()


@pytest.mark.parametrize("dt", DTS, ids=IDS)
@pytest.mark.parametrize("nseq, lo, hi, lq, heads, d, page", [
    (1, 3000, 3000, 1, (8, 2), 64, 64), (1, 9000, 9000, 3, (4, 4), 128, 256), (5, 0, 2500, 2, (16, 4), 32, 16),
    (70, 0, 1500, 1, (2, 1), 64, 32), (2, 600, 5000, 1, (6, 1), 256, 128), (2, 600, 2000, 1, (3, 3), 96, 16)])
def test_cut_keys(nseq, lo, hi, lq, heads, d, page, dt):
    r = random.Random(nseq)
    lens = [hi] + [r.randint(lo, hi) for _ in range(nseq - 1)]
    if nseq > 3:
        lens[1], lens[2] = 0, 1
    c = Case(nseq + d, [lq] * nseq, lens, *heads, d, dt, page=page)
    assert c.spec().plan().parts > 1
    c.check()


@pytest.mark.parametrize("max_len", [1, 600, 100000])
def test_any_lengths_whatever_was_foreseen(max_len):
    c = Case(3, [1, 2, 40], [2500, 7, 1200], 8, 2, 64, DType.BF16, page=16)
    c.check(spec=c.spec(max_len=max_len))


@pytest.mark.parametrize("dt", DTS, ids=IDS)
def test_pages_outside_the_cache_hold_no_keys(dt):
    c = Case(4, [1, 3, 20], [100, 64, 20], 4, 2, 64, dt)
    c.table[0, 2], c.table[0, 6], c.table[1, :4], c.table[2, 0] = -1, c.pages, -7, 1 << 30
    c.check()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [32, 96, 128, 256])
def test_nan_keys_and_values_reach_the_rows_that_see_them(d, causal):
    c = Case(5, [40, 1, 9], [100, 70, 9], 4, 2, d, DType.F16, causal=causal)
    for b, j, head, block, which in [(0, 90, 0, 0, 1), (0, 95, 1, d // 32 - 1, 0), (1, 3, 0, d // 32 - 1, 1), (2, 8, 1, 0, 1)]:
        c.cache[2 * which + 1][c.table[b, j // 16], head, j % 16, block] = 255
    want, _ = c.want()
    assert torch.isnan(want).any() and not torch.isnan(want).all()
    c.check()


def test_lengths_past_the_table_and_starts_past_the_rows():
    c = Case(6, [2, 2], [64, 64], 4, 2, 64, DType.F32, extra=0)
    out = torch.full((4, c.qw), -9.0, device=DEV)
    spec = c.spec(table_width=4)
    cache = [x.to(DEV) for x in c.cache]
    table = c.table[:, :4].contiguous().to(DEV)
    spec.run(c.q.to(DEV), *cache, i32([0, 2, 90]), table, i32([64, 1000]), out)
    good = c.run(c.spec())
    assert torch.equal(out.cpu().view(4, 4, 64), good)
    out.fill_(-9.0)
    spec.run(c.q.to(DEV), *cache, i32([0, 2, 2]), table, i32([64, -5]), out)
    assert torch.equal(out[:2].cpu().view(2, 4, 64), good[:2]) and (out[2:] == -9).all()
    # no pages at all: no keys
    c.spec(table_width=4, pages=0).run(c.q.to(DEV), None, None, None, None, i32([0, 2, 4]), None, i32([64, 64]), out)
    assert (out == 0).all()


def test_large_and_tiny_scores():
    for scale in (1e-20, 3.0, 1e4, 1e10):
        c = Case(7, [3, 1], [200, 333], 4, 2, 64, DType.F32, scale=scale)
        got = c.run().double()
        want, _ = c.want()
        assert torch.isfinite(got).all()
        if scale < 1:
            c.check(got)
        elif scale > 100:  # one key has all of it, unless two are as near as a rounding
            assert ((got - want).abs().amax(-1) < 1e-3).double().mean() > 0.95


def test_infinite_queries():
    c = Case(8, [1, 1, 1], [50, 50, 50], 2, 1, 64, DType.F32)
    c.q[1, :64] = float("nan")
    c.q[2, 64 + 5] = float("inf")
    got = c.run()
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1, 0]).all() and torch.isfinite(got[1, 1]).all()
    assert torch.isfinite(got[2, 0]).all() and torch.isnan(got[2, 1]).all()


def test_cache_beyond_4_gib():
    # one page table entry in the last pages of a cache whose codes pass 2^32 bytes
    hkv, d, page = 8, 256, 4096
    pages = (1 << 32) // (hkv * page * d // 2) + 2
    cache = mx4.kv4_cache(pages, page, hkv, d)
    x = torch.randn(5, 4 * hkv + 2 * hkv, d, device=DEV).bfloat16()
    slots = [(pages - 1) * page + 7 + i for i in range(5)]
    q = torch.empty(5, 4 * hkv, d, dtype=torch.bfloat16, device=DEV)
    mx4.Kv4AppendSpec(tokens=5, hq=4 * hkv, hkv=hkv, d=d, page=page, pages=pages, dt=DType.BF16).run(
        x, None, None, None, None, None, i32(slots), q, *cache)
    small = mx4.kv4_cache(1, page, hkv, d)
    for a, b in zip(small, cache):
        a.copy_(b[-1:])
    assert (small[1][0, :, 7:12] > 0).all()
    out, ref = torch.empty_like(q), torch.empty_like(q)
    for c, n, o in ((cache, pages, out), (small, 1, ref)):
        mx4.Kv4AttnSpec(nseq=1, tokens=5, hq=4 * hkv, hkv=hkv, d=d, page=page, pages=n, table_width=1, dt=DType.BF16).run(
            q, *c, i32([0, 5]), i32([n - 1]), i32([12]), o)
    assert torch.equal(out, ref) and torch.isfinite(out).all()


@pytest.mark.parametrize("lens", [[40, 300, 1], [1500, 2600, 900]])
def test_captured_replays_follow_lengths_and_tables(lens):
    c = Case(9, [1] * 3, lens, 8, 2, 64, DType.F16, page=16)
    cache = [x.to(DEV) for x in c.cache]
    spec = c.spec()
    n = spec.workspace_bytes()
    ws = torch.empty(n // 4 + 1, device=DEV)
    q, q_start, k_len, table = c.q.to(DEV), i32(c.q_start), i32(lens), c.table.to(DEV)
    out = torch.empty(3, c.qw, dtype=torch.float16, device=DEV)
    run = lambda: spec.run(q, *cache, q_start, table, k_len, out, ws=ws)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        k_len.copy_(i32([max(0, x - 37 * i) for x in lens]))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        run()
        assert torch.equal(got, out) and torch.isfinite(got).all()


def test_two_streams_with_a_workspace_each():
    c = Case(10, [1, 1], [3000, 2000], 8, 2, 128, DType.BF16, page=64)
    want = c.run()
    cache = [x.to(DEV) for x in c.cache]
    spec, q, q_start, table, k_len = c.spec(), c.q.to(DEV), i32(c.q_start), c.table.to(DEV), i32(c.k_lens)
    outs = [torch.empty(2, c.qw, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for s, o in zip(streams, outs):
            spec.run(q, *cache, q_start, table, k_len, o, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu().view_as(want), want) for o in outs)


def test_append_then_attend_as_a_stream_grows():
    # one token at a time into shared pages, against the same keys at once
    hq, hkv, d, page, n, dt = 4, 2, 64, 16, 40, DType.BF16
    g = torch.Generator().manual_seed(11)
    x = torch.randn(n, 2, hq + 2 * hkv, d, generator=g).to(TORCH[dt]).to(DEV)  # two streams
    cos, sin = rotation_tables(n, d, device=DEV)
    table = i32([[5, 1, 3], [0, 4, 2]])
    cache, whole = mx4.kv4_cache(6, page, hkv, d), mx4.kv4_cache(6, page, hkv, d)
    spec = dict(hq=hq, hkv=hkv, d=d, page=page, pages=6, dt=dt)
    q, out = torch.empty(2, 2, hq, d, dtype=TORCH[dt], device=DEV)
    last = []
    for t in range(n):
        pos = i32([t, t])
        slots = table[:, t // page] * page + t % page
        mx4.Kv4AppendSpec(tokens=2, rot=d, positions=n, **spec).run(x[t], None, None, cos, sin, pos, slots, q, *cache)
        mx4.Kv4AttnSpec(nseq=2, tokens=2, table_width=3, **spec).run(q, *cache, i32([0, 1, 2]), table, i32([t + 1, t + 1]), out)
        last.append(out.clone())
    xs = x.transpose(0, 1).reshape(2 * n, hq + 2 * hkv, d).contiguous()
    t = torch.arange(n, device=DEV)
    slots = (table[:, t // page] * page + t % page).flatten().int()
    q, out = torch.empty(2, 2 * n, hq, d, dtype=TORCH[dt], device=DEV)
    mx4.Kv4AppendSpec(tokens=2 * n, rot=d, positions=n, **spec).run(xs, None, None, cos, sin, t.repeat(2).int(), slots, q, *whole)
    mx4.Kv4AttnSpec(nseq=2, tokens=2 * n, table_width=3, **spec).run(q, *whole, i32([0, n, 2 * n]), table, i32([n, n]), out)
    for a, b in zip(cache, whole):
        assert torch.equal(a, b)
    steps = torch.stack(last).transpose(0, 1).reshape(2 * n, hq, d)
    # the same sums in another order and with other maxima: two roundings of a probability and one of the result
    assert (steps.float() - out.float()).abs().max() <= 4 * 2.0 ** -8 * out.float().abs().max()


def test_short_strided_and_other_tensors_are_refused():
    c = Case(12, [1], [20], 4, 2, 64, DType.F16)
    cache = [x.to(DEV) for x in c.cache]
    args = dict(q=c.q.to(DEV), k_codes=cache[0], k_scales=cache[1], v_codes=cache[2], v_scales=cache[3], q_start=i32([0, 1]),
                table=c.table.to(DEV), k_len=i32([20]), out=torch.empty(1, c.qw, dtype=torch.float16, device=DEV))
    spec = c.spec()
    spec.run(*args.values())
    for name, t in args.items():
        for bad in (t.flatten()[:-1], t.double(), t.cpu()):
            with pytest.raises(AihError, match=f"{name} must be a dense tensor"):
                spec.run(*{**args, name: bad}.values())


@pytest.mark.parametrize("norm", [False, True])
def test_a_captured_step_follows_positions_and_slots(norm):
    # one token of four streams: into the cache and attention over it, replayed with other rows each time
    hq, hkv, d, page, dt, n = 8, 2, 64, 16, DType.BF16, 60
    g = torch.Generator().manual_seed(13)
    cos, sin = rotation_tables(n, d, device=DEV)
    table = torch.randperm(16, generator=g).int().view(4, 4).to(DEV)
    caches = [mx4.kv4_cache(16, page, hkv, d) for _ in range(2)]
    w = (1 + 0.1 * torch.randn(d, generator=g)).to(TORCH[dt]).to(DEV) if norm else None
    append = mx4.Kv4AppendSpec(tokens=4, hq=hq, hkv=hkv, d=d, page=page, pages=16, rot=d, positions=n, norm=norm, dt=dt)
    attn = mx4.Kv4AttnSpec(nseq=4, tokens=4, hq=hq, hkv=hkv, d=d, page=page, pages=16, table_width=4, dt=dt)
    x = torch.empty(4, hq + 2 * hkv, d, dtype=TORCH[dt], device=DEV)
    pos, slots, k_len = (torch.zeros(4, dtype=torch.int32, device=DEV) for _ in range(3))
    q_start = i32([0, 1, 2, 3, 4])
    q, out = torch.empty(2, 4, hq, d, dtype=TORCH[dt], device=DEV)

    def step(cache):
        append.run(x, w, w, cos, sin, pos, slots, q, *cache)
        attn.run(q, *cache, q_start, table, k_len, out)

    slots.fill_(-1)
    step(caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(caches[0])
    for t in range(40):
        at = torch.tensor([t, t // 2, t, 59 - t])
        x.copy_(torch.randn(4, hq + 2 * hkv, d, generator=g))
        pos.copy_(at.int()), k_len.copy_((at + 1).int())
        slots.copy_(table[torch.arange(4), at.to(DEV) // page] * page + at.to(DEV) % page)
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        step(caches[1])
        assert torch.equal(out, replayed) and torch.isfinite(out).all()
    for a, b in zip(*caches):
        assert torch.equal(a, b)


def test_appending_on_another_stream_and_into_a_slice_of_a_projection():
    hq, hkv, d = 2, 1, 96
    x = torch.randn(90, 2 * hq + 2 * hkv, d, device=DEV)
    cos, sin = rotation_tables(90, d, device=DEV)
    slots = torch.arange(90, dtype=torch.int32, device=DEV)
    spec = dict(tokens=90, hq=hq, hkv=hkv, d=d, rot=d, positions=90, page=32, pages=3)
    own, other = mx4.kv4_cache(3, 32, hkv, d), mx4.kv4_cache(3, 32, hkv, d)
    q = torch.empty(2, 90, hq, d, device=DEV)
    dense = x[:, hq:].contiguous()
    mx4.Kv4AppendSpec(**spec).run(dense, None, None, cos, sin, None, slots, q[0], *own)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    row = x.shape[1] * d
    at = x.data_ptr() + hq * d * 4  # the heads from hq on, still in the projection's rows
    mx4.Kv4AppendSpec(**spec, x_stride=row).run(at, None, None, cos, sin, None, slots, q[1], *other, stream=s)
    s.synchronize()
    assert torch.equal(q[0], q[1]) and all(torch.equal(a, b) for a, b in zip(own, other))
