"""GPU tests of the attention operators against plain 64-bit computations.

Tolerances are worst-case bounds, per element, of what the kernels round; u is
2^-24, w the storage type's unit roundoff (2^-24, 2^-11, 2^-8 for f32, f16,
bf16).

Attention: a score's error is at most ds = scale (d + 8) u max_j sum|q||k| plus the
rounding of the exponent's argument, 4 u max|s|; a probability is then off by a
factor of 1 +- 2 (ds + 8 u), rounded to the storage type (w; an absolute 2^-32 of
the largest in f16, whose probabilities go down to subnormals), and the sums of
n products add n u each. With A_i = sum_j p_ij |v_j| / sum_j p_ij,
  |o - exact| <= A (4 ds + w + (2 n + 64) u) + w |exact| + n 2^-32 max|v| + tiny,
tiny one subnormal step of the storage type.

Norm and rotation: the mean square of d values is off by (d + 4) u, its inverse
root by half of it and two roundings, and a rotated value is a sum of two
products: |y - exact| <= (|a| + |b|)((d + 16) u) + w |exact| + tiny.
"""
import math

import numpy as np
import pytest
import torch

from ai_engine_amd import attn
from ai_engine_amd.conv import DType

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TORCH = {DType.F32: torch.float32, DType.F16: torch.float16, DType.BF16: torch.bfloat16}
U = 2.0 ** -24
W = {DType.F32: 2.0 ** -24, DType.F16: 2.0 ** -11, DType.BF16: 2.0 ** -8}
TINY = {DType.F32: 1e-38, DType.F16: 2.0 ** -24, DType.BF16: 1e-38}
ALL = [DType.F32, DType.F16, DType.BF16]


def rnd(gen, *shape, dt, scale=1.0):
    return (torch.randn(*shape, generator=gen, dtype=torch.float32) * scale).to(TORCH[dt])


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts(ls):
    return [0, *np.cumsum(ls).tolist()]


class Case:
    """Packed sequences on the host, with the 64-bit result and its bound."""

    def __init__(self, dt, hq, hkv, d, q_lens, k_lens, causal=True, scale=None, prefix=0, seed=0, gap=0, kscale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dt, self.hq, self.hkv, self.d, self.causal, self.scale = dt, hq, hkv, d, causal, scale
        self.q_lens, self.k_lens, self.prefix = q_lens, k_lens, prefix
        self.q_starts = starts(q_lens)
        self.k_starts = [s + gap * (i + 1) for i, s in enumerate(starts(k_lens)[:-1])]
        self.tokens, self.rows = self.q_starts[-1], sum(k_lens) + gap * (len(k_lens) + 1)
        self.q = rnd(g, self.tokens, hq, d, dt=dt, scale=kscale)
        self.k, self.v = rnd(g, self.rows, hkv, d, dt=dt, scale=kscale), rnd(g, self.rows, hkv, d, dt=dt)
        self.pk, self.pv = rnd(g, prefix, hkv, d, dt=dt), rnd(g, prefix, hkv, d, dt=dt)

    def spec(self, **kw):
        return attn.AttnSpec(**{**dict(nseq=len(self.q_lens), tokens=self.tokens, rows=self.rows, hq=self.hq,
                                       hkv=self.hkv, d=self.d, causal=self.causal, scale=self.scale, dt=self.dt,
                                       max_len=max(self.k_lens, default=0), prefix=self.prefix), **kw})

    def run(self, spec=None, out=None, q=None, k=None, v=None, **kw):
        spec = spec or self.spec()
        if out is None:
            out = torch.full((self.tokens, self.hq, self.d), float("nan"), dtype=TORCH[self.dt], device=DEV)
        dev = lambda t, o: o if o is not None else t.to(DEV)
        spec.run(dev(self.q, q), dev(self.k, k), dev(self.v, v), i32(self.q_starts), i32(self.k_starts),
                 i32(self.k_lens), out, prefix_k=self.pk.to(DEV) if self.prefix else None,
                 prefix_v=self.pv.to(DEV) if self.prefix else None, **kw)
        torch.cuda.synchronize()
        return out.cpu()

    def exact(self):
        """(o, bound), both [tokens, hq, d] in 64 bits."""
        scale = self.scale if self.scale is not None else 1.0 / math.sqrt(self.d)
        o = torch.zeros(self.tokens, self.hq, self.d, dtype=torch.float64)
        e = torch.zeros_like(o)
        for b, (lq, lk) in enumerate(zip(self.q_lens, self.k_lens)):
            for i in range(lq):
                seen = max(0, min(lk, i + 1 + lk - lq)) if self.causal else lk
                k0 = self.k_starts[b]
                kk = torch.cat([self.pk, self.k[k0:k0 + seen]]).double()
                vv = torch.cat([self.pv, self.v[k0:k0 + seen]]).double()
                t = self.q_starts[b] + i
                n = kk.shape[0]
                if n == 0:
                    continue
                q = self.q[t].double().view(self.hkv, -1, self.d)              # [hkv, g, d]
                kk, vv = kk.transpose(0, 1), vv.transpose(0, 1)                # [hkv, n, d]
                s = scale * q @ kk.transpose(1, 2)                             # [hkv, g, n]
                p = torch.softmax(s, -1)
                ds = scale * (self.d + 8) * U * (q.abs() @ kk.abs().transpose(1, 2)).amax(-1, keepdim=True)
                ds = ds + 4 * U * s.abs().amax(-1, keepdim=True)
                oo = p @ vv
                a = p @ vv.abs()
                w = W[self.dt]
                err = a * (4 * ds + w + (2 * n + 64) * U) + w * oo.abs() + n * 2.0 ** -32 * vv.abs().max() + TINY[self.dt]
                o[t], e[t] = oo.reshape(self.hq, self.d), err.reshape(self.hq, self.d)
        return o, e

    def check(self, got=None, **kw):
        got = self.run(**kw) if got is None else got
        o, e = self.exact()
        bad = ~((got.double() - o).abs() <= e)
        assert not bad.any(), (int(bad.sum()), float(((got.double() - o).abs() / e).max()))
        return got


# ---------------------------------------------------------------- attention: sizes, types, heads

@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [8, 32, 40, 64, 72, 96, 128, 136, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_head_sizes(dt, d, causal):
    lens = [1, 33, 70, 129]
    Case(dt, 4, 2, d, lens, lens, causal, seed=d).check()


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [8, 32, 56, 64, 96, 128, 200, 256])
def test_single_token_head_sizes(dt, d):
    k_lens = [1, 31, 32, 33, 300, 127, 129, 0]
    c = Case(dt, 6, 2, d, [1] * 8, k_lens, seed=d, gap=3)
    assert c.spec().plan().kernel == attn.AttnKernel.KEYS
    got = c.check()
    assert (got[7] == 0).all()


@pytest.mark.parametrize("hq, hkv", [(1, 1), (5, 5), (7, 1), (6, 3), (24, 8), (32, 1), (40, 1)])
@pytest.mark.parametrize("lq", [1, 3])
def test_grouped_heads(hq, hkv, lq):
    lens = [200, 45, 4]
    Case(DType.F16, hq, hkv, 64, [lq] * 3, lens, seed=hq, gap=1).check()
    Case(DType.BF16, hq, hkv, 32, [40, 3, 77], [40, 90, 77], seed=hq).check()


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 257])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_lengths(n, causal):
    Case(DType.F16, 2, 1, 64, [n], [n], causal, seed=n).check()
    Case(DType.BF16, 3, 3, 128, [n, n + 1], [n + 5, n], causal, seed=n).check()


@pytest.mark.parametrize("dt", ALL)
def test_rows_without_keys(dt):
    # more queries than keys: the first rows see nothing; empty sequences in
    # between, with and without queries
    c = Case(dt, 4, 2, 64, [50, 0, 7, 3, 0, 40], [20, 9, 0, 1, 0, 39], seed=1)
    got = c.check()
    assert (got[:30] == 0).all() and (got[50:57] == 0).all()
    c = Case(dt, 4, 2, 64, [5, 1, 4], [2, 0, 1], seed=2)
    assert c.spec().plan().kernel == attn.AttnKernel.KEYS
    assert (c.check()[:3] == 0).all()


def test_no_keys_at_all():
    c = Case(DType.F16, 4, 2, 64, [1, 2], [0, 0])
    spec = c.spec()
    out = torch.full((3, 4, 64), float("nan"), dtype=torch.float16, device=DEV)
    spec.run(c.q.to(DEV), None, None, i32([0, 1, 3]), i32([0, 0]), i32([0, 0]), out)
    assert (out.cpu() == 0).all()


def test_many_sequences():
    r = np.random.default_rng(5)
    lens = r.integers(0, 9, 300).tolist()
    Case(DType.F16, 2, 1, 32, lens, lens, seed=3).check()
    Case(DType.F16, 4, 1, 32, [1] * 300, lens, seed=4).check()


@pytest.mark.parametrize("scale", [0.01, 1.0, 3.7])
@pytest.mark.parametrize("dt", ALL)
def test_scale(dt, scale):
    Case(dt, 2, 2, 32, [60], [60], scale=scale, seed=9).check()


@pytest.mark.parametrize("dt", ALL)
def test_large_scores(dt):
    # scores of several thousand: one key takes all, nothing overflows
    c = Case(dt, 2, 1, 64, [70, 1], [70, 90], scale=1.0, kscale=25.0, seed=4)
    got = c.run()
    o, e = c.exact()
    assert torch.isfinite(got).all()
    assert ((got.double() - o).abs() <= e).all()


# ---------------------------------------------------------------- keys cut into parts

@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("lens", [[1300, 256, 257], [1023, 0, 2049], [3000, 1, 513]])
def test_cut_keys(dt, lens):
    c = Case(dt, 4, 2, 64, [1] * 3, lens, seed=6)
    p = c.spec(max_len=3000).plan()
    assert p.parts > 1
    c.check(spec=c.spec(max_len=3000))


@pytest.mark.parametrize("hint", [1, 300, 999, 5000, 2 ** 31 - 1])
def test_length_hint_is_only_a_hint(hint):
    c = Case(DType.F16, 4, 2, 64, [1, 1], [1500, 700], seed=7)
    c.check(spec=c.spec(max_len=hint))


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("causal", [True, False])
def test_few_rows_after_a_long_past(dt, causal):
    # a chunk of a prompt: tiles of rows whose keys are cut
    c = Case(dt, 4, 2, 64, [40], [1700], causal, seed=8)
    assert c.spec().plan().parts > 1
    c.check()


# ---------------------------------------------------------------- shared prefix

@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("prefix", [1, 64, 700])
@pytest.mark.parametrize("lq", [1, 4])
def test_prefix(dt, prefix, lq):
    Case(dt, 8, 2, 64, [lq] * 5, [0, 1, 3, 40, 130], prefix=prefix, seed=prefix + lq).check()


@pytest.mark.parametrize("d", [40, 96, 128, 256])
def test_prefix_head_sizes(d):
    Case(DType.BF16, 4, 1, d, [1] * 20, list(range(20)), prefix=333, seed=d).check()


def test_prefix_behind_prompts():
    Case(DType.F16, 4, 2, 64, [60, 0, 130], [60, 5, 200], prefix=90, seed=3).check()
    Case(DType.F16, 4, 2, 64, [60, 9], [60, 12], causal=False, prefix=90, seed=4).check()


# ---------------------------------------------------------------- what is not seen

@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
def test_unseen_keys_do_not_leak(dt, bad, d):
    # a bad key and value at one position: rows before it come out as with
    # zeros there, rows from it on do not stay finite
    n, at = 150, 77
    c = Case(dt, 2, 1, d, [n], [n], seed=11)
    c.k[at], c.v[at] = 0, 0
    want = c.run()
    c.v[at] = bad
    c.v[at, :, 5] = 0
    got = c.run()
    assert torch.equal(got[:at], want[:at])
    seen = torch.ones(d, dtype=torch.bool)
    seen[5] = False
    assert not torch.isfinite(got[at:][..., seen]).any()
    assert torch.equal(got[at:][..., 5], want[at:][..., 5])
    c.k[at] = bad
    assert torch.equal(c.run()[:at], want[:at])


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("lq", [1, 3])
def test_rows_past_the_length_do_not_leak(dt, lq):
    c = Case(dt, 4, 2, 64, [lq] * 3, [37, 3, 290], gap=40, seed=12)
    want = c.run()
    for t in (c.k, c.v):
        keep = t.clone()
        t[:] = float("nan")
        for s, n in zip(c.k_starts, c.k_lens):
            t[s:s + n] = keep[s:s + n]
    assert torch.equal(c.run(), want)


@pytest.mark.parametrize("dt", ALL)
def test_few_queries_with_a_bad_last_value(dt):
    # three tokens over a cache, the newest value not finite: only the newest
    # token sees it
    c = Case(dt, 4, 2, 64, [3], [100], seed=13)
    c.v[99] = 0
    want = c.run()
    c.v[99] = float("inf")
    got = c.run()
    assert torch.equal(got[:2], want[:2]) and not torch.isfinite(got[2]).any()


def test_a_bad_query_stays_its_own():
    c = Case(DType.F16, 2, 1, 64, [90], [90], seed=14)
    want = c.run()
    c.q[40] = float("nan")
    got = c.run()
    rest = torch.arange(90) != 40
    assert torch.equal(got[rest], want[rest]) and torch.isnan(got[40]).all()


# ---------------------------------------------------------------- memory: strides, bounds, offsets

@pytest.mark.parametrize("dt", ALL)
def test_strided_rows(dt):
    # q, k and v inside the projection's rows, the output inside wider rows
    lens = [70, 33]
    c = Case(dt, 4, 2, 64, lens, lens, seed=15)
    n = c.tokens
    wide = torch.full((n, 4 + 2 + 2 + 1, 64), float("nan"), dtype=TORCH[dt], device=DEV)
    wide[:, :4], wide[:, 4:6], wide[:, 6:8] = c.q.to(DEV), c.k.to(DEV), c.v.to(DEV)
    out = torch.full((n, 6, 64), 3.0, dtype=TORCH[dt], device=DEV)
    s = 9 * 64
    spec = c.spec(q_stride=s, k_stride=s, v_stride=s, o_stride=6 * 64)
    c.run(spec=spec, out=out, q=wide, k=wide[:, 4:], v=wide[:, 6:])
    c.check(got=out[:, :4].cpu())
    assert (out[:, 4:] == 3.0).all()


def test_strided_prefix():
    c = Case(DType.F16, 4, 2, 64, [1] * 3, [9, 0, 40], prefix=100, seed=16)
    both = torch.cat([c.pk, c.pv], 1).to(DEV)
    spec = c.spec(pk_stride=256, pv_stride=256)
    out = torch.full((3, 4, 64), float("nan"), dtype=torch.float16, device=DEV)
    spec.run(c.q.to(DEV), c.k.to(DEV), c.v.to(DEV), i32(c.q_starts), i32(c.k_starts), i32(c.k_lens), out,
             prefix_k=both, prefix_v=both[:, 2:])
    c.check(got=out.cpu())


def test_starts_and_lengths_past_the_tensors_are_cut():
    c = Case(DType.F16, 4, 2, 64, [3, 4], [10, 12], seed=17)
    out = torch.full((7, 4, 64), float("nan"), dtype=torch.float16, device=DEV)
    args = [t.to(DEV) for t in (c.q, c.k, c.v)]
    c.spec().run(*args, i32([0, 3, 99]), i32([0, 10]), i32([10, 10 ** 9]), out)
    c.check(got=out.cpu())
    c.spec().run(*args, i32([-5, 3, 7]), i32([-3, 10]), i32([10, 12]), out)
    c.check(got=out.cpu())
    c.spec().run(*args, i32([0, 3, 7]), i32([0, 10 ** 9]), i32([10, 12]), out)
    assert (out[3:] == 0).all()
    c.spec().run(*args, i32([0, 3, 7]), i32([0, 10]), i32([10, -1]), out)
    assert (out[3:] == 0).all()


def test_rows_of_no_sequence_are_not_written():
    c = Case(DType.F16, 4, 2, 64, [40, 30], [40, 30], seed=18)
    out = torch.full((100, 4, 64), 5.0, dtype=torch.float16, device=DEV)
    q = torch.zeros(100, 4, 64, dtype=torch.float16)
    q[10:80] = c.q
    spec = c.spec(tokens=100)
    spec.run(q.to(DEV), c.k.to(DEV), c.v.to(DEV), i32([10, 50, 80]), i32(c.k_starts), i32(c.k_lens), out)
    c.check(got=out[10:80].cpu())
    assert (out[:10] == 5.0).all() and (out[80:] == 5.0).all()


@pytest.mark.parametrize("prefix", [0, 700])
@pytest.mark.parametrize("lq", [1, 40])
def test_rows_of_no_sequence_are_not_written_by_a_join(prefix, lq):
    lens = [3000, 1, 1500]
    c = Case(DType.F16, 4, 2, 64, [lq] * 3, lens, prefix=prefix, seed=19)
    out = torch.full((c.tokens + 30, 4, 64), 5.0, dtype=torch.float16, device=DEV)
    q = torch.ones(c.tokens + 30, 4, 64, dtype=torch.float16)
    q[10:-20] = c.q
    spec = c.spec(tokens=c.tokens + 30)
    assert spec.workspace_bytes() > 0
    ws = torch.ones(spec.workspace_bytes() // 4, device=DEV)
    spec.run(q.to(DEV), c.k.to(DEV), c.v.to(DEV), i32([10 + s for s in c.q_starts]), i32(c.k_starts), i32(c.k_lens),
             out, prefix_k=c.pk.to(DEV) if prefix else None, prefix_v=c.pv.to(DEV) if prefix else None, ws=ws)
    c.check(got=out[10:-20].cpu())
    assert (out[:10] == 5.0).all() and (out[-20:] == 5.0).all()


@pytest.mark.parametrize("lq", [1, 40])
def test_a_cache_beyond_32_bit_offsets(lq):
    # 2^31 elements and 4 GiB lie before the sequence's rows
    hkv, d, n = 8, 128, 300
    c = Case(DType.F16, 16, hkv, d, [lq], [n], seed=19)
    rows = (1 << 32) // (2 * hkv * d) + n + 7
    k = torch.zeros(rows, hkv, d, dtype=torch.float16, device=DEV)
    v = torch.zeros(rows, hkv, d, dtype=torch.float16, device=DEV)
    k0 = rows - n
    k[k0:], v[k0:] = c.k.to(DEV), c.v.to(DEV)
    out = torch.full((lq, 16, d), float("nan"), dtype=torch.float16, device=DEV)
    c.spec(rows=rows).run(c.q.to(DEV), k, v, i32([0, lq]), i32([k0]), i32([n]), out)
    c.check(got=out.cpu())


# ---------------------------------------------------------------- blocks, orders and cuts

@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("d", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_that_end_inside_a_stage(dt, d, causal):
    # ends in the first and the second half of a stage, wavefronts without rows
    k_lens = [1, 32, 33, 64, 65, 96, 97, 130, 161]
    Case(dt, 2, 1, d, [70] * len(k_lens), k_lens, causal, seed=d + 1).check()


@pytest.mark.parametrize("n", [2, 31, 32, 33])
@pytest.mark.parametrize("dt", [DType.F16, DType.F32])
def test_sequences_in_any_order(n, dt):
    r = np.random.default_rng(n)
    lens = r.integers(0, 60, n).tolist()
    lens[0], lens[-1] = 0, 75  # an empty one, the longest last, some equal
    Case(dt, 4, 2, 64, lens, lens, seed=n).check()
    Case(dt, 2, 1, 128, [max(1, v // 2) for v in lens], lens, False, seed=n + 1, gap=1).check()


def test_the_order_changes_nothing():
    lens = [40, 7, 130, 0, 64, 130]
    a = Case(DType.BF16, 4, 2, 64, lens, lens, seed=31)
    want = a.run()
    at = starts(lens)
    for order in ([5, 4, 3, 2, 1, 0], [2, 0, 5, 1, 4, 3]):
        b = Case(DType.BF16, 4, 2, 64, [lens[i] for i in order], [lens[i] for i in order], seed=32)
        rows = torch.cat([torch.arange(at[i], at[i + 1]) for i in order])
        b.q, b.k, b.v = a.q[rows], a.k[rows], a.v[rows]
        assert torch.equal(b.run(), want[rows])


@pytest.mark.parametrize("d", [72, 96, 128, 256])
@pytest.mark.parametrize("lens", [[129], [300, 131, 0], [1000, 128, 257]])
def test_fp32_keys_over_more_wavefronts_and_parts(d, lens):
    Case(DType.F32, 4, 2, d, [1] * len(lens), lens, seed=d).check()
    Case(DType.F32, 2, 2, d, [20] * len(lens), lens, seed=d + 1).check()


@pytest.mark.parametrize("dt, kernel", [(DType.F16, attn.AttnKernel.ROWS), (DType.F32, attn.AttnKernel.KEYS)])
def test_a_long_prefix_under_many_rows(dt, kernel):
    # 16 bit: much to read for every 32 rows, so in a launch of its own
    c = Case(dt, 8, 1, 32, [1] * 512, [5, 0, 9, 2] * 128, prefix=8200, seed=41)
    p = c.spec().plan()
    assert (p.kernel, p.prefix_kernel) == (attn.AttnKernel.KEYS, kernel) and p.prefix_parts > 1
    c.check()


# ---------------------------------------------------------------- calls

@pytest.mark.parametrize("kind", ["prompt", "cut", "prefix"])
def test_same_bits_every_time(kind):
    if kind == "prompt":
        c = Case(DType.BF16, 8, 2, 128, [300, 77], [300, 77], seed=20)
    elif kind == "cut":
        c = Case(DType.F16, 8, 2, 64, [1] * 4, [5000, 3000, 10, 0], seed=21)
    else:
        c = Case(DType.F32, 8, 2, 64, [2] * 9, list(range(9)), prefix=900, seed=22)
    want = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), want)


def test_on_another_stream_and_with_its_own_workspace():
    c = Case(DType.F16, 8, 2, 64, [1] * 4, [5000, 3000, 10, 0], seed=23)
    want = c.run()
    spec = c.spec()
    ws = torch.full((spec.workspace_bytes() // 4,), float("nan"), device=DEV)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    args = [t.to(DEV) for t in (c.q, c.k, c.v)] + [i32(c.q_starts), i32(c.k_starts), i32(c.k_lens)]
    out = torch.full((4, 8, 64), float("nan"), dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    spec.run(*args, out, ws=ws, stream=st)
    st.synchronize()
    assert torch.equal(out.cpu(), want)
    with torch.cuda.stream(st):
        out.fill_(float("nan"))
        spec.run(*args, out, ws=ws)
    st.synchronize()
    assert torch.equal(out.cpu(), want)


def test_raw_addresses():
    c = Case(DType.F16, 8, 2, 64, [1] * 4, [5000, 3000, 10, 0], seed=23)
    spec = c.spec()
    args = [t.to(DEV) for t in (c.q, c.k, c.v)] + [i32(c.q_starts), i32(c.k_starts), i32(c.k_lens)]
    out = torch.full((4, 8, 64), float("nan"), dtype=torch.float16, device=DEV)
    assert spec.workspace_bytes() > 0
    spec.run(*[t.data_ptr() for t in args], out.data_ptr())
    c.check(got=out.cpu())


@pytest.mark.parametrize("raw", [False, True])
def test_a_workspace_made_by_the_call_belongs_to_its_stream(raw):
    c = Case(DType.F16, 8, 2, 64, [1] * 4, [5000, 3000, 10, 0], seed=23)
    want = c.run()
    spec = c.spec()
    args = [t.to(DEV) for t in (c.q, c.k, c.v)] + [i32(c.q_starts), i32(c.k_starts), i32(c.k_lens)]
    out = torch.full((4, 8, 64), float("nan"), dtype=torch.float16, device=DEV)
    n = spec.workspace_bytes() // 4
    a = torch.randn(4096, 4096, device=DEV)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(8):  # keeps the stream busy while the host goes on
            a @ a
    spec.run(*args, out, stream=st.cuda_stream if raw else st)
    others = [torch.full((n,), 7.0, device=DEV) for _ in range(3)]  # on the current stream, at once
    torch.cuda.synchronize()
    assert torch.equal(out.cpu(), want)
    assert all(bool((o == 7.0).all()) for o in others)


def test_graph_replay():
    c = Case(DType.F16, 8, 2, 64, [1] * 4, [5000, 3000, 10, 0], prefix=200, seed=24)
    spec = c.spec()
    ws = torch.empty(spec.workspace_bytes() // 4, device=DEV)
    args = [t.to(DEV) for t in (c.q, c.k, c.v)] + [i32(c.q_starts), i32(c.k_starts), i32(c.k_lens)]
    kw = dict(prefix_k=c.pk.to(DEV), prefix_v=c.pv.to(DEV), ws=ws)
    out = torch.empty(4, 8, 64, dtype=torch.float16, device=DEV)
    spec.run(*args, out, **kw)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        spec.run(*args, out, **kw)
    for step in range(4):
        # new inputs and lengths in the same buffers, as a serving loop has them
        args[0].mul_(0.9)
        args[5].copy_(i32([5000 - step, 3000 - 700 * step, 10 + step, step]))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(float("nan"))
        spec.run(*args, out, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, out) and torch.isfinite(got).all()


# ---------------------------------------------------------------- norms and rotation

class Rope:
    def __init__(self, dt, tokens, hq, hkv, d, rot, pairs=False, npos=50, seed=0, wide=0, eps=1e-6, scale=2.0):
        g = torch.Generator().manual_seed(seed)
        self.dt, self.tokens, self.hq, self.hkv, self.d, self.rot, self.pairs = dt, tokens, hq, hkv, d, rot, pairs
        self.eps, self.npos, self.wide = eps, npos, wide
        self.x = rnd(g, tokens, hq + 2 * hkv + wide, d, dt=dt, scale=scale)
        self.wq, self.wk = 1 + rnd(g, d, dt=dt, scale=0.3), 1 + rnd(g, d, dt=dt, scale=0.3)
        ang = torch.rand(npos, max(rot // 2, 1), generator=g, dtype=torch.float64) * 6.3
        self.cos, self.sin = ang.cos().float(), ang.sin().float()
        self.pos = torch.randint(0, npos, (tokens,), generator=g).to(torch.int32)

    def spec(self, **kw):
        return attn.QkNormRopeSpec(**{**dict(tokens=self.tokens, hq=self.hq, hkv=self.hkv, d=self.d, rot=self.rot,
                                             pairs=self.pairs, eps=self.eps, dt=self.dt, positions=self.npos,
                                             x_stride=(self.hq + 2 * self.hkv + self.wide) * self.d), **kw})

    def exact(self, weights=True, pos=None):
        """(q, k, v) and the bounds of q and k."""
        pos = (self.pos if pos is None else pos).long()
        x = self.x.double()
        out, err = [], []
        for part, w in ((x[:, :self.hq], self.wq), (x[:, self.hq:self.hq + self.hkv], self.wk)):
            y = part / torch.sqrt((part * part).mean(-1, keepdim=True) + self.eps)
            if weights:
                y = y * w.double()
            m = y.abs()
            if self.rot:
                c, s = self.cos[pos].double()[:, None], self.sin[pos].double()[:, None]
                h = self.rot // 2
                ia = 2 * torch.arange(h) if self.pairs else torch.arange(h)
                ib = ia + (1 if self.pairs else h)
                a, b = y[..., ia], y[..., ib]
                y, m = y.clone(), m.clone()
                y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
                m[..., ia] = m[..., ib] = a.abs() + b.abs()
            out.append(y)
            err.append(m * (self.d + 16) * U + W[self.dt] * y.abs() + TINY[self.dt])
        return out, x[:, self.hq + self.hkv:self.hq + 2 * self.hkv], err

    def buffers(self, rows=None, fill=float("nan")):
        rows = self.tokens if rows is None else rows
        new = lambda n, h: torch.full((n, h, self.d), fill, dtype=TORCH[self.dt], device=DEV)
        return new(self.tokens, self.hq), new(rows, self.hkv), new(rows, self.hkv)

    def run(self, spec=None, weights=True, pos="own", slots=None, bufs=None, v=True):
        q, k, vv = bufs or self.buffers()
        pos = self.pos.to(DEV) if isinstance(pos, str) else pos
        (spec or self.spec()).run(self.x.to(DEV), self.wq.to(DEV) if weights else None,
                                  self.wk.to(DEV) if weights else None, self.cos.to(DEV), self.sin.to(DEV), pos,
                                  slots, q, k, vv if v else None)
        torch.cuda.synchronize()
        return q.cpu(), k.cpu(), vv.cpu()

    def check(self, got, weights=True, pos=None):
        (q, k), v, (eq, ek) = self.exact(weights, pos)
        assert ((got[0].double() - q).abs() <= eq).all()
        assert ((got[1].double() - k).abs() <= ek).all()
        if got[2] is not None:
            assert torch.equal(got[2].double(), v)


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("d, rot", [(8, 0), (8, 4), (8, 8), (32, 32), (40, 20), (40, 40), (64, 32), (72, 68), (96, 48),
                                    (128, 128), (200, 12), (256, 252), (256, 256)])
def test_rope_head_sizes(dt, pairs, d, rot):
    r = Rope(dt, 13, 5, 2, d, rot, pairs, seed=d + rot)
    r.check(r.run())


@pytest.mark.parametrize("dt", ALL)
@pytest.mark.parametrize("tokens, hq, hkv", [(1, 1, 1), (1, 32, 8), (257, 3, 1), (65, 7, 7), (5, 1, 0), (1000, 8, 2)])
def test_rope_rows_and_heads(dt, tokens, hq, hkv):
    r = Rope(dt, tokens, hq, hkv, 64, 64, seed=tokens)
    r.check(r.run())


@pytest.mark.parametrize("dt", ALL)
def test_rope_without_weights_positions_values(dt):
    r = Rope(dt, 50, 4, 2, 64, 64, npos=50, seed=2)
    r.check(r.run(weights=False), weights=False)
    r.check(r.run(pos=None), pos=torch.arange(50))
    q, k, v = r.run(v=False)
    r.check((q, k, None))
    assert torch.isnan(v).all()


def test_rope_positions_outside_the_tables_take_the_nearest_row():
    r = Rope(DType.F32, 6, 2, 1, 32, 32, npos=9, seed=3)
    pos = torch.tensor([-1, 0, 8, 9, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    r.check(r.run(pos=pos.to(DEV)), pos=pos.clamp(0, 8))


@pytest.mark.parametrize("dt", ALL)
def test_rope_into_cache_rows(dt):
    # tokens without a row, and rows outside the cache: dropped
    r = Rope(dt, 9, 4, 2, 64, 64, seed=4)
    slots = [5, -1, 0, 19, 20, 2 ** 31 - 1, -2 ** 31, 7, 3]
    bufs = r.buffers(rows=20, fill=4.0)
    q, k, v = r.run(spec=r.spec(rows=20), slots=i32(slots), bufs=bufs)
    (wq, wk), wv, (eq, ek) = r.exact()
    assert ((q.double() - wq).abs() <= eq).all()
    used = {s: t for t, s in enumerate(slots) if 0 <= s < 20}
    for row in range(20):
        if row in used:
            t = used[row]
            assert ((k[row].double() - wk[t]).abs() <= ek[t]).all() and torch.equal(v[row].double(), wv[t])
        else:
            assert (k[row] == 4.0).all() and (v[row] == 4.0).all()


def test_rope_fewer_rows_than_tokens_without_slots():
    r = Rope(DType.F16, 9, 4, 2, 64, 64, seed=5)
    bufs = r.buffers(rows=6)
    q, k, v = r.run(spec=r.spec(rows=6), bufs=bufs)
    (wq, wk), wv, (eq, ek) = r.exact()
    assert ((q.double() - wq).abs() <= eq).all() and ((k.double() - wk[:6]).abs() <= ek[:6]).all()
    assert torch.equal(v.double(), wv[:6])


@pytest.mark.parametrize("dt", ALL)
def test_rope_strides_and_in_place(dt):
    r = Rope(dt, 33, 4, 2, 64, 64, seed=6, wide=1)
    x = r.x.to(DEV)
    s = 9 * 64
    keep = x.clone()
    r.spec(q_stride=s, k_stride=s, v_stride=s).run(x, r.wq.to(DEV), r.wk.to(DEV), r.cos.to(DEV), r.sin.to(DEV),
                                                   r.pos.to(DEV), None, x, x[:, 4:], None)
    torch.cuda.synchronize()
    r.check((x[:, :4].cpu(), x[:, 4:6].cpu(), None))
    assert torch.equal(x[:, 6:].cpu(), keep[:, 6:].cpu())


@pytest.mark.parametrize("dt", ALL)
def test_rope_zero_and_non_finite_heads(dt):
    r = Rope(dt, 4, 2, 1, 64, 64, seed=7)
    r.x[0, 0] = 0
    r.x[1, 1, 3] = float("nan")
    r.x[2, 3, 9] = float("inf")  # a value head: copied as it is
    q, k, v = r.run()
    assert (q[0, 0] == 0).all()
    assert torch.isnan(q[1, 1]).all() and torch.isfinite(q[1, 0]).all() and torch.isfinite(k).all()
    assert torch.equal(v, r.x[:, 3:])


def test_rope_rows_beyond_32_bit_offsets():
    d, hkv = 256, 8
    rows = (1 << 32) // (4 * hkv * d) + 5
    r = Rope(DType.F32, 3, 2, hkv, d, 256, seed=8)
    k = torch.zeros(rows, hkv, d, device=DEV)
    v = torch.zeros(rows, hkv, d, device=DEV)
    slots = [rows - 1, 1, rows - 3]
    q = torch.empty(3, 2, d, device=DEV)
    r.run(spec=r.spec(rows=rows), slots=i32(slots), bufs=(q, k, v))
    idx = torch.tensor(slots, device=DEV)
    r.check((q.cpu(), k[idx].cpu(), v[idx].cpu()))
    assert int(torch.count_nonzero(k).item()) <= 3 * hkv * d and (k[0] == 0).all() and (k[2] == 0).all()
