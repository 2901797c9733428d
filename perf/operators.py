"""The timed attention operators: what a user of this framework runs between the
two pointwise convs of an attention block, over the sizes and types they run it
with.

A case is a dict of plain values whose "kind" names the operator:
  rope    head norms of queries and keys with the position rotation, in one
          pass from the projection's rows; keys and values go to their cache
          rows when the case has a cache
  prompt  attention over whole prompts: packed sequences of different lengths,
          grouped heads, causal or not, optionally after `past` earlier keys
  cache   attention of `lq` tokens per sequence over each sequence's cache
  prefix  the same, behind `prefix` keys that the whole batch shares

Lengths are drawn from the case's own `lens` number, so they belong to the case
and not to the inputs' seed.  With `own` false, `run` computes the plain form
in fp32 torch operations; with `own` true it calls ai_engine_amd.attn.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NBYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


# ---------------------------------------------------------------- the cases

def _rope(name, tokens, hq, hkv, d, rot, dt, pairs=False, cap=0, skip=False):
    c = dict(name=name) if name else {}
    return c | dict(kind="rope", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, pairs=pairs, cap=cap, skip=skip, dt=dt)


def _prompt(name, nseq, lo, hi, hq, hkv, d, dt, causal=True, past=0, lens=0):
    c = dict(name=name) if name else {}
    return c | dict(kind="prompt", nseq=nseq, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, causal=causal, past=past, lens=lens,
                    dt=dt)


def _cache(name, nseq, lo, hi, hq, hkv, d, dt, lq=1, lens=0):
    c = dict(name=name) if name else {}
    return c | dict(kind="cache", nseq=nseq, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, lq=lq, lens=lens, dt=dt)


def _prefix(name, nseq, prefix, lo, hi, hq, hkv, d, dt, lq=1, lens=0):
    c = dict(name=name) if name else {}
    return c | dict(kind="prefix", nseq=nseq, prefix=prefix, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, lq=lq, lens=lens,
                    dt=dt)


def listed():
    return [
        # one step of a small serving batch: eight new tokens into the cache,
        # where the launch is all the cost
        _rope("rope_8tok_cache_bf16", 8, 32, 8, 128, 128, "bf16", cap=8192),
        # the tokens of 64 frames at 20 x 36 after their QKV projection
        _rope("rope_64x20x36_f16", 64 * 20 * 36, 8, 2, 64, 64, "f16"),
        # three short prompts, one of a single token: the smallest prompt call
        _prompt("prompt_3x1to180_f16", 3, 1, 180, 8, 8, 32, "f16", lens=5),
        # every token of a 20 x 36 frame sees its whole frame, 64 frames
        _prompt("prompt_64x20x36_full_f16", 64, 720, 720, 8, 2, 64, "f16", causal=False),
        # prompts of a serving batch, packed, of very different lengths
        _prompt("prompt_24ragged_bf16", 24, 60, 2500, 32, 8, 128, "bf16", lens=1),
        # one long prompt
        _prompt("prompt_16384_bf16", 1, 16384, 16384, 32, 8, 128, "bf16"),
        # fp32, the storage type of the shipped models, odd lengths and a head
        # size that is no power of two
        _prompt("prompt_7odd_f32", 7, 181, 1441, 8, 4, 96, "f32", lens=2),
        # one stream's next token over the 180 tokens of a 10 x 18 frame:
        # latency
        _cache("cache_b1_180_f32", 1, 180, 180, 8, 2, 64, "f32"),
        # a serving batch at very different positions, an empty and a
        # one-token cache among them
        _cache("cache_b64_ragged_bf16", 64, 0, 8192, 32, 8, 128, "bf16", lens=3),
        # one very long stream: the keys have to be split to fill the chip
        _cache("cache_b1_131071_f16", 1, 131071, 131071, 16, 4, 128, "f16"),
        # a batch that answers from one shared context
        _prefix("prefix_b64_4096_bf16", 64, 4096, 1, 512, 32, 8, 128, "bf16", lens=4),
        # a few streams with two tokens each behind a frame's 720 tokens
        _prefix("prefix_b6_720_f16", 6, 720, 9, 77, 8, 2, 64, "f16", lq=2, lens=6),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


# what a drawn case may cost: the largest listed one's work, with the fp32
# matrix rate a sixteenth of the 16-bit one
_MAX_FLOPS = {"f32": 1.3e11, "f16": 2.2e12, "bf16": 2.2e12}
_MAX_BYTES = 8.0e8
_MAX_HELD = 2.5e9  # a cache's whole region, used or not


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        rows = c["nseq"] * c["hi"] if c["kind"] in ("cache", "prefix") else c.get("cap", 0)
        if 2 * rows * c["hkv"] * c["d"] * NBYTES[c["dt"]] > _MAX_HELD:
            continue
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_FLOPS[c["dt"]]:
            return c


def _draw(rng):
    kind = rng.choice(["rope", "prompt", "prompt", "cache", "cache", "prefix"])
    dt = rng.choice(["f32", "f16", "f16", "bf16", "bf16"])
    d = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 256])
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 4, 6, 8])
    lens = rng.randrange(1 << 20)
    if kind == "rope":
        tokens = _logint(rng, 1, 65536)
        cap = rng.choice([0, _logint(rng, tokens, 4 * tokens + 64)])
        return _rope(None, tokens, hq, hkv, d, rng.choice([d, d, d // 2, 0]), dt, pairs=rng.random() < 0.4, cap=cap,
                     skip=cap > 0 and rng.random() < 0.5)
    if kind == "prompt":
        hi = _logint(rng, 16, 16384)
        nseq = _logint(rng, 1, max(1, min(64, 65536 // hi)))
        past = rng.choice([0, 0, _logint(rng, 1, 4096)])
        return _prompt(None, nseq, max(1, hi // rng.choice([1, 4, 64])), hi, hq, hkv, d, dt,
                       causal=rng.random() < 0.7, past=past, lens=lens)
    if kind == "cache":
        hi = _logint(rng, 16, 131072)
        nseq = _logint(rng, 1, 128)
        return _cache(None, nseq, rng.choice([0, hi // 8, hi]), hi, hq, hkv, d, dt, lq=rng.choice([1, 1, 1, 2, 5]),
                      lens=lens)
    hi = _logint(rng, 16, 2048)
    return _prefix(None, _logint(rng, 2, 128), _logint(rng, 32, 32768), rng.choice([0, 1, hi]), hi, hq, hkv, d, dt,
                   lq=rng.choice([1, 1, 2, 4]), lens=lens)


def _lengths(case):
    """The sequences' lengths: spread over [lo, hi] by their logarithm, the
    first one hi; with lo = 0 also an empty one and a single token."""
    lo, hi, n = case["lo"], case["hi"], case["nseq"]
    r = random.Random(case["lens"])
    out = [_logint(r, max(lo, 1), hi) for _ in range(n)]
    if lo == 0 and n >= 3:
        out[1], out[2] = 0, 1
    elif lo == 1 and n >= 3:
        out[1] = 1
    out[0] = hi
    return out


def _pairs(case):
    """(query, key) pairs per head, and the key rows read."""
    ls = _lengths(case)
    if case["kind"] == "prompt":
        past = case["past"]
        pairs = sum(l * (l + 1) // 2 + l * past if case["causal"] else l * (l + past) for l in ls)
        return pairs, sum(ls), sum(l + past for l in ls)
    lq = case["lq"]
    pre = case.get("prefix", 0)
    # the queries are each sequence's last lq tokens
    pairs = sum(max(0, l - lq + 1 + i) for l in ls for i in range(lq)) + pre * lq * case["nseq"]
    return pairs, lq * case["nseq"], sum(ls) + pre


def work(case):
    e, d = NBYTES[case["dt"]], case["d"]
    hq, hkv = case["hq"], case["hkv"]
    if case["kind"] == "rope":
        n = case["tokens"] * (hq + 2 * hkv) * d
        table = case["tokens"] * (case["rot"] * 4 + 4)  # the rows of the tables that the positions name
        return {"bytes": 2 * n * e + table + 2 * d * e + (4 * case["tokens"] if case["cap"] else 0),
                "flops": case["tokens"] * (hq + hkv) * (4 * d + 3 * case["rot"])}
    pairs, nq, nk = _pairs(case)
    return {"bytes": 2 * nq * hq * d * e + 2 * nk * hkv * d * e, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------- inputs

def _normal(gen, shape, dt, scale=1.0):
    """Seeded N(0, scale^2), made in pieces so that large inputs need no
    large fp32 temporary."""
    out = torch.empty(shape, dtype=TORCH[dt], device=DEV)
    flat = out.view(-1)
    step = 1 << 26
    for o in range(0, flat.numel(), step):
        n = min(step, flat.numel() - o)
        flat[o:o + n] = torch.randn(n, generator=gen, device=DEV, dtype=torch.float32) * scale
    return out


def _starts(ls):
    out = [0]
    for l in ls:
        out.append(out[-1] + l)
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = _prepare_rope(case, gen) if case["kind"] == "rope" else _prepare_attn(case, gen)
    st["case"] = case
    if own:
        _prepare_own(st)
    return st


def _prepare_rope(case, gen):
    t, hq, hkv, d, rot, dt = (case[k] for k in ("tokens", "hq", "hkv", "d", "rot", "dt"))
    st = {"x": _normal(gen, (t, (hq + 2 * hkv) * d), dt, 1.7)}
    st["wq"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)).to(TORCH[dt])
    st["wk"] = (1.0 + 0.2 * torch.randn(d, generator=gen, device=DEV)).to(TORCH[dt])
    npos = max(t, 4096)
    st["pos"] = torch.randint(0, npos, (t,), generator=gen, device=DEV, dtype=torch.int32)
    half = max(rot // 2, 1)
    freq = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    ang = torch.arange(npos, device=DEV, dtype=torch.float64)[:, None] * freq
    st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
    rows = case["cap"] or t
    st["slots"] = None
    if case["cap"]:
        slots = torch.randperm(rows, generator=gen, device=DEV)[:t].to(torch.int32)
        if case["skip"]:  # padding tokens, which have no cache row
            slots[torch.rand(t, generator=gen, device=DEV) < 0.1] = -1
        st["slots"] = slots
    st["q"] = torch.zeros(t, hq, d, dtype=TORCH[dt], device=DEV)
    st["k"] = _normal(gen, (rows, hkv, d), dt) if case["cap"] else torch.zeros(rows, hkv, d, dtype=TORCH[dt], device=DEV)
    st["v"] = _normal(gen, (rows, hkv, d), dt) if case["cap"] else torch.zeros(rows, hkv, d, dtype=TORCH[dt], device=DEV)
    return st


def _prepare_attn(case, gen):
    hq, hkv, d, dt = (case[k] for k in ("hq", "hkv", "d", "dt"))
    ls = _lengths(case)
    st = {}
    if case["kind"] == "prompt":
        past = case["past"]
        q_lens, k_lens = ls, [l + past for l in ls]
        k_starts = _starts(k_lens)[:-1]
        rows = sum(k_lens)
    else:
        # one region of `hi` rows a sequence, filled up to its length
        q_lens, k_lens = [case["lq"]] * case["nseq"], ls
        k_starts = [b * case["hi"] for b in range(case["nseq"])]
        rows = case["nseq"] * case["hi"]
    q_starts = _starts(q_lens)
    t = q_starts[-1]
    st["q"] = _normal(gen, (t, hq, d), dt)
    if case["kind"] == "prompt" and case["past"] == 0:
        # values stay in the projection's rows, as one piece of each
        st["k"] = _normal(gen, (rows, hkv, d), dt)
        st["qkv"] = _normal(gen, (rows, hq + 2 * hkv, d), dt)
        st["v"] = st["qkv"][:, hq + hkv:]
    else:
        st["k"] = _normal(gen, (rows, hkv, d), dt)
        st["v"] = _normal(gen, (rows, hkv, d), dt)
    if case["kind"] == "prefix":
        st["pk"] = _normal(gen, (case["prefix"], hkv, d), dt)
        st["pv"] = _normal(gen, (case["prefix"], hkv, d), dt)
    st["scale"] = 1.0 / math.sqrt(d)
    st["q_lens"], st["k_lens"], st["q_starts"], st["k_starts"] = q_lens, k_lens, q_starts, k_starts
    st["q_start"], st["k_start"], st["k_len"] = _i32(q_starts), _i32(k_starts), _i32(k_lens)
    st["causal"] = case.get("causal", True)
    st["rows"] = rows
    return st


# ---------------------------------------------------------------- the framework's calls

def _prepare_own(st):
    from ai_engine_amd import attn, conv

    c = st["case"]
    dt = {"f32": conv.DType.F32, "f16": conv.DType.F16, "bf16": conv.DType.BF16}[c["dt"]]
    if c["kind"] == "rope":
        st["spec"] = attn.QkNormRopeSpec(tokens=c["tokens"], hq=c["hq"], hkv=c["hkv"], d=c["d"], rot=c["rot"],
                                         pairs=c["pairs"], eps=EPS, dt=dt, positions=st["cos"].shape[0],
                                         rows=st["k"].shape[0])
        return
    st["spec"] = attn.AttnSpec(nseq=c["nseq"], tokens=st["q_starts"][-1], rows=st["rows"], hq=c["hq"], hkv=c["hkv"],
                               d=c["d"], causal=st["causal"], scale=st["scale"], dt=dt, v_stride=st["v"].stride(0),
                               max_len=max(st["k_lens"]), prefix=c.get("prefix", 0))
    st["out"] = torch.zeros(st["q_starts"][-1], c["hq"], c["d"], dtype=TORCH[c["dt"]], device=DEV)
    n = st["spec"].workspace_bytes()
    st["ws"] = torch.zeros(n // 4, dtype=torch.float32, device=DEV) if n else None


def run(state):
    if own:
        if state["case"]["kind"] == "rope":
            state["spec"].run(state["x"], state["wq"], state["wk"], state["cos"], state["sin"], state["pos"],
                              state["slots"], state["q"], state["k"], state["v"])
            return state["q"], state["k"], state["v"]
        state["spec"].run(state["q"], state["k"], state["v"], state["q_start"], state["k_start"], state["k_len"],
                          state["out"], prefix_k=state.get("pk"), prefix_v=state.get("pv"), ws=state["ws"])
        return state["out"]
    if state["case"]["kind"] == "rope":
        return _plain_rope(state)
    return _plain_attn(state)


# ---------------------------------------------------------------- the plain forms, fp32

def _plain_rope(st):
    c = st["case"]
    t, hq, hkv, d, rot = c["tokens"], c["hq"], c["hkv"], c["d"], c["rot"]
    x = st["x"].view(t, hq + 2 * hkv, d)
    h = rot // 2
    cos, sin = st["cos"][st["pos"].long()][:, None], st["sin"][st["pos"].long()][:, None]

    def norm_rotate(y, w):
        y = y.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        if rot == 0:
            return y
        r, rest = y[..., :rot], y[..., rot:]
        if c["pairs"]:
            a, b = r[..., 0::2], r[..., 1::2]
            out = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = r[..., :h], r[..., h:]
            out = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([out, rest], -1)

    q = norm_rotate(x[:, :hq], st["wq"]).to(x.dtype)
    k = norm_rotate(x[:, hq:hq + hkv], st["wk"]).to(x.dtype)
    v = x[:, hq + hkv:]
    if st["slots"] is None:
        return q, k, v.contiguous()
    # the cache with one row more, which takes the tokens without a row
    rows = st["k"].shape[0]
    to = torch.where(st["slots"] < 0, rows, st["slots"]).long()
    kc = torch.cat([st["k"], st["k"][:1]])
    vc = torch.cat([st["v"], st["v"][:1]])
    kc[to] = k
    vc[to] = v
    return q, kc[:rows], vc[:rows]


_SCORES = 1 << 29  # fp32 scores held at once


def _plain_seq(q, k, v, scale, own_keys, causal):
    """q [Lq, Hq, D] against k, v [Lk, Hkv, D]: the last `own_keys` keys are
    under the causal mask, the ones before them seen by all."""
    lq, hq, d = q.shape
    lk, hkv, _ = k.shape
    if lk == 0 or lq == 0:
        return torch.zeros(lq, hq, d, dtype=q.dtype, device=q.device)
    g = hq // hkv
    qh = (q.float() * scale).permute(1, 0, 2).reshape(hkv, g * lq, d)
    kh = k.float().permute(1, 2, 0).contiguous()
    vh = v.float().permute(1, 0, 2).contiguous()
    hidden = None
    if causal:
        i = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
        j = torch.arange(lk, device=q.device)[None]
        hidden = (j > i) & (j >= lk - own_keys)
    out = torch.empty(hkv, g * lq, d, device=q.device)
    step = max(1, _SCORES // (g * lq * lk))
    for a in range(0, hkv, step):
        s = torch.matmul(qh[a:a + step], kh[a:a + step])
        if hidden is not None:
            s = s.view(-1, g, lq, lk).masked_fill(hidden, float("-inf")).view(-1, g * lq, lk)
        m = s.amax(-1, keepdim=True)
        m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        out[a:a + step] = torch.matmul(p, vh[a:a + step]) / torch.where(z == 0, torch.ones_like(z), z)
    return out.view(hkv, g, lq, d).permute(2, 0, 1, 3).reshape(lq, hq, d).to(q.dtype)


def _plain_attn(st):
    outs = []
    for b, (lq, lk) in enumerate(zip(st["q_lens"], st["k_lens"])):
        q0, k0 = st["q_starts"][b], st["k_starts"][b]
        k, v = st["k"][k0:k0 + lk], st["v"][k0:k0 + lk]
        if "pk" in st:
            k, v = torch.cat([st["pk"], k]), torch.cat([st["pv"], v])
        outs.append(_plain_seq(st["q"][q0:q0 + lq], k, v, st["scale"], lk, st["causal"]))
    return torch.cat(outs)


# ---------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(st)
    return _exact_attn(st)


def _exact_rope(st):
    c = st["case"]
    t, hq, hkv, d, rot = c["tokens"], c["hq"], c["hkv"], c["d"], c["rot"]
    heads = hq + 2 * hkv
    x = st["x"].double().reshape(t, heads, d)
    out = torch.empty_like(x)
    out[:, hq + hkv:] = x[:, hq + hkv:]
    # the rotation as a complex product, dim by dim pairs
    i = torch.arange(rot // 2, device=DEV)
    first, second = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + rot // 2)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()]
    for h in range(hq + hkv):
        y = x[:, h]
        w = (st["wq"] if h < hq else st["wk"]).double()
        y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / d + EPS) * w
        if rot:
            z = torch.complex(y[:, first].contiguous(), y[:, second].contiguous()) * turn
            y[:, first], y[:, second] = z.real, z.imag
        out[:, h] = y
    k, v = out[:, hq:hq + hkv], out[:, hq + hkv:]
    if st["slots"] is not None:
        kc, vc = st["k"].double(), st["v"].double()
        for j, row in enumerate(st["slots"].tolist()) if t <= 64 else ():
            if row >= 0:
                kc[row], vc[row] = k[j], v[j]
        if t > 64:
            keep = torch.nonzero(st["slots"] >= 0).flatten()
            kc.index_copy_(0, st["slots"][keep].long(), k[keep])
            vc.index_copy_(0, st["slots"][keep].long(), v[keep])
        k, v = kc, vc
    return out[:, :hq].contiguous(), k.contiguous(), v.contiguous()


def _exact_attn(st):
    c = st["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    out = torch.zeros(st["q_starts"][-1], hq, d, dtype=torch.float64, device=DEV)
    pre = c.get("prefix", 0)
    for b in range(c["nseq"]):
        lq, lk, q0, k0 = st["q_lens"][b], st["k_lens"][b], st["q_starts"][b], st["k_starts"][b]
        if lq == 0 or lk + pre == 0:
            continue
        for h in range(hkv):
            k, v = st["k"][k0:k0 + lk, h].double(), st["v"][k0:k0 + lk, h].double()
            if pre:
                k, v = torch.cat([st["pk"][:, h].double(), k]), torch.cat([st["pv"][:, h].double(), v])
            kt = k.t().contiguous()
            # blocks of query rows, each against the keys that its last row sees
            for hh in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                for r0 in range(0, lq, 4096):
                    r1 = min(lq, r0 + 4096)
                    seen = torch.full((r1 - r0,), lk, device=DEV)
                    if st["causal"]:
                        seen = torch.arange(r0, r1, device=DEV) + (lk - lq) + 1
                    seen = seen.clamp(min=0) + pre
                    n = max(0, (r1 + lk - lq) if st["causal"] else lk) + pre
                    if n == 0:
                        continue
                    s = st["q"][q0 + r0:q0 + r1, hh].double() @ kt[:, :n].contiguous() * st["scale"]
                    s[torch.arange(n, device=DEV)[None] >= seen[:, None]] = -math.inf
                    lse = torch.logsumexp(s, -1, keepdim=True)
                    p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse))
                    out[q0 + r0:q0 + r1, hh] = p @ v[:n]
    return out
