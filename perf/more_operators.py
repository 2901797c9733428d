"""The timed 4-bit operators: rows held in microscaled 4-bit floating point (blocks
of 32 elements with one power-of-two scale), the pointwise product of such rows,
and a paged cache of keys and values in the same format with its attention.

A case is a dict of plain values whose "kind" names the operators:
  round   rows to 4 bits and back: what is stored, and the values it stands for
  linear  a pointwise conv in 4 bits: the activations' quantisation and the
          product with weights that were quantised when they were loaded, with
          the bias, the activation and the residual
  append  rotation of queries and keys and the new keys' and values' way into
          the pages of a 4-bit cache; the cache is read back as values
  attn    attention over such a cache: `lq` tokens of every sequence, or whole
          prompts behind `past` earlier keys

Lengths and page orders are drawn from the case's own `lens` number, so they
belong to the case and not to the inputs' seed.  With `own` false, `run`
computes the plain form in fp32 torch operations; with `own` true it calls
ai_engine_amd.mx4.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
NBYTES = {"f32": 4, "f16": 2, "bf16": 2}
BITS4 = 17 / 32  # bytes an element: a code and its share of the block's scale


# ---------------------------------------------------------------- the cases

def _round(name, rows, k, dt):
    c = dict(name=name) if name else {}
    return c | dict(kind="round", rows=rows, k=k, dt=dt)


def _linear(name, m, k, cout, dt, act="none", residual=False):
    c = dict(name=name) if name else {}
    return c | dict(kind="linear", m=m, k=k, cout=cout, act=act, residual=residual, dt=dt)


def _append(name, tokens, hq, hkv, d, rot, dt, page=64, cap=0, pairs=False, skip=False):
    c = dict(name=name) if name else {}
    return c | dict(kind="append", tokens=tokens, hq=hq, hkv=hkv, d=d, rot=rot, page=page, cap=cap, pairs=pairs, skip=skip,
                    dt=dt)


def _attn(name, nseq, lo, hi, hq, hkv, d, dt, lq=1, past=None, page=64, causal=True, lens=0):
    """lq tokens a sequence over lo..hi keys each; with `past`, prompts of lo..hi tokens behind `past` keys each."""
    c = dict(name=name) if name else {}
    return c | dict(kind="attn", nseq=nseq, lo=lo, hi=hi, hq=hq, hkv=hkv, d=d, lq=lq, past=past, page=page, causal=causal,
                    lens=lens, dt=dt)


def listed():
    return [
        # the activations of a few tokens: the launches are all the cost
        _round("round_9x4096_bf16", 9, 4096, "bf16"),
        # the activations of 256 frames at 10 x 18 x 960
        _round("round_256x10x18x960_f16", 256 * 180, 960, "f16"),
        # one step of a serving batch of eight through a square projection
        _linear("linear_8x4096x4096_bf16", 8, 4096, 4096, "bf16"),
        # the encoder's long 1x1 conv, 256 frames of 10 x 18, with its
        # activation and a residual
        _linear("linear_256x10x18_960x160_f16", 256 * 180, 960, 160, "f16", act="relu6", residual=True),
        # sizes that fill no tile, fp32, the storage type of the shipped models
        _linear("linear_1007x1000x724_f32", 1007, 1000, 724, "f32", act="hardswish"),
        # the largest: a whole prompt batch through a square projection
        _linear("linear_8192x8192x8192_bf16", 8192, 8192, 8192, "bf16"),
        # eight new tokens of a serving batch into pages of 64 rows
        _append("append_8tok_bf16", 8, 32, 8, 128, 128, "bf16", cap=512),
        # the tokens of 64 frames at 20 x 36, adjacent pairs rotated
        _append("append_64x20x36_f16", 64 * 720, 8, 2, 64, 64, "f16", cap=64 * 768, pairs=True),
        # one stream's next token over the 180 tokens of a 10 x 18 frame:
        # latency
        _attn("attn_b1_180_f32", 1, 180, 180, 8, 2, 64, "f32"),
        # a serving batch at very different positions, an empty and a
        # one-token cache among them
        _attn("attn_b64_ragged_bf16", 64, 0, 8192, 32, 8, 128, "bf16", lens=3),
        # one very long stream: the keys have to be split to fill the chip
        _attn("attn_b1_131071_f16", 1, 131071, 131071, 16, 4, 128, "f16", page=256),
        # new prompts of different lengths behind what their streams hold
        _attn("attn_4prompts_past2000_bf16", 4, 100, 1024, 32, 8, 128, "bf16", past=2000, lens=2),
    ]


def _logint(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


# what a drawn case may cost: the largest listed one's work
_MAX_FLOPS = {"linear": 1.09e12, "attn": 2.0e11}
_MAX_BYTES = 4.0e8
_MAX_SCORES = 4.0e8  # of the plain form, padded: what it has to hold at once


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        if w["bytes"] > _MAX_BYTES or w["flops"] > _MAX_FLOPS.get(c["kind"], 1e18):
            continue
        if c["kind"] == "attn":
            longest = c["hi"] + (c["past"] or 0)
            rows = c["lq"] if c["past"] is None else c["hi"]
            if c["nseq"] * rows * c["hq"] * longest > _MAX_SCORES or c["nseq"] * longest * c["hkv"] * c["d"] > 1.5e9:
                continue
        return c


def _draw(rng):
    kind = rng.choice(["round", "linear", "linear", "append", "attn", "attn"])
    dt = rng.choice(["f32", "f16", "f16", "bf16", "bf16"])
    if kind == "round":
        return _round(None, _logint(rng, 1, 65536), 4 * _logint(rng, 1, 2048), dt)
    if kind == "linear":
        return _linear(None, _logint(rng, 1, 65536), 4 * _logint(rng, 8, 2048), 4 * _logint(rng, 1, 2048), dt,
                       act=rng.choice(["none", "none", "relu", "relu6", "hardswish"]), residual=rng.random() < 0.4)
    d = rng.choice([32, 64, 64, 96, 128, 128, 128, 192, 256])
    hkv = rng.choice([1, 2, 3, 4, 8])
    hq = hkv * rng.choice([1, 2, 3, 4, 4, 6, 8])
    page = rng.choice([16, 32, 64, 64, 128, 256])
    if kind == "append":
        tokens = _logint(rng, 1, 65536)
        cap = -(-_logint(rng, tokens, 3 * tokens + 64) // page) * page
        return _append(None, tokens, hq, hkv, d, rng.choice([d, d, d // 2, 0]), dt, page=page, cap=cap,
                       pairs=rng.random() < 0.4, skip=rng.random() < 0.4)
    lens = rng.randrange(1 << 20)
    if rng.random() < 0.4:
        hi = _logint(rng, 16, 4096)
        return _attn(None, _logint(rng, 1, 32), max(1, hi // rng.choice([1, 4, 64])), hi, hq, hkv, d, dt,
                     past=rng.choice([0, _logint(rng, 1, 8192)]), page=page, causal=rng.random() < 0.7, lens=lens)
    hi = _logint(rng, 16, 131072)
    return _attn(None, _logint(rng, 1, 128), rng.choice([0, hi // 8, hi]), hi, hq, hkv, d, dt,
                 lq=rng.choice([1, 1, 1, 2, 5]), page=page, lens=lens)


def _lengths(case):
    """The sequences' lengths: spread over [lo, hi] by their logarithm, the
    first one hi; with lo = 0 also an empty one and a single token."""
    lo, hi, n = case["lo"], case["hi"], case["nseq"]
    r = random.Random(case["lens"])
    out = [_logint(r, max(lo, 1), hi) for _ in range(n)]
    if lo == 0 and n >= 3:
        out[1], out[2] = 0, 1
    out[0] = hi
    return out


def _q_k_lengths(case):
    ls = _lengths(case)
    if case["past"] is None:
        return [case["lq"]] * case["nseq"], ls
    return ls, [n + case["past"] for n in ls]


def work(case):
    e = NBYTES[case["dt"]]
    if case["kind"] == "round":
        n = case["rows"] * case["k"]
        return {"bytes": n * (2 * e + BITS4), "flops": 2 * n}
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["cout"]
        return {"bytes": m * k * e + n * k * BITS4 + m * n * e * (2 if case["residual"] else 1) + n * e,
                "flops": 2 * m * k * n}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "append":
        t, held = case["tokens"], 2 * case["cap"] * hkv * d
        table = t * (case["rot"] * 4 + 8) if case["rot"] else 4 * t
        return {"bytes": t * d * ((hq + 2 * hkv) * e + hq * e + 2 * hkv * BITS4) + table + held * (BITS4 + e),
                "flops": t * (hq + hkv) * 3 * case["rot"] + held}
    q_lens, k_lens = _q_k_lengths(case)
    pairs = sum(sum(min(lk, max(0, lk - lq + 1 + i)) for i in range(lq)) if case["causal"] else lq * lk
                for lq, lk in zip(q_lens, k_lens))
    return {"bytes": 2 * sum(q_lens) * hq * d * e + 2 * sum(k_lens) * hkv * d * BITS4, "flops": 4 * pairs * hq * d}


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


def _uneven(gen, rows, k, dt):
    """Rows whose channels are of different size, as activations are."""
    size = torch.exp(torch.randn(k, generator=gen, device=DEV))
    return (_normal(gen, (rows, k), "f32") * size).to(TORCH[dt])


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    st = {"round": _prepare_round, "linear": _prepare_linear, "append": _prepare_append,
          "attn": _prepare_attn}[case["kind"]](case, gen)
    st["case"] = case
    if own:
        _prepare_own(st)
    return st


def _prepare_round(case, gen):
    return {"x": _uneven(gen, case["rows"], case["k"], case["dt"])}


def _padded(k):
    return -(-k // 128) * 128


def _scale_bytes(k):
    """A row's scales, in whole 16s."""
    return -(-k // 512) * 16


def _prepare_linear(case, gen):
    m, k, n, dt = (case[i] for i in ("m", "k", "cout", "dt"))
    st = {"x": _uneven(gen, m, k, dt)}
    # the weights as a loader keeps them: in 4 bits
    st["w_codes"], st["w_scales"] = _plain_quant(_normal(gen, (n, k), dt, 1 / math.sqrt(k)))
    st["bias"] = _normal(gen, (n,), dt, 0.1)
    st["res"] = _normal(gen, (m, n), dt) if case["residual"] else None
    return st


def _tables(positions, rot):
    half = max(rot // 2, 1)
    freq = 10000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
    ang = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * freq
    return ang.cos().float(), ang.sin().float()


def _random_cache(gen, rows, d):
    """rows of d values of N(0, 1) in 4 bits, made in pieces."""
    codes = torch.empty(rows, d // 2, dtype=torch.uint8, device=DEV)
    scales = torch.empty(rows, d // 32, dtype=torch.uint8, device=DEV)
    step = (1 << 24) // d
    for r in range(0, rows, step):
        n = min(step, rows - r)
        codes[r:r + n], scales[r:r + n] = _quant_blocks(torch.randn(n, d // 32, 32, generator=gen, device=DEV))
    return codes, scales


def _prepare_append(case, gen):
    t, hq, hkv, d, page, cap, dt = (case[i] for i in ("tokens", "hq", "hkv", "d", "page", "cap", "dt"))
    st = {"x": _normal(gen, (t, hq + 2 * hkv, d), dt, 1.7)}
    npos = max(t, 4096)
    st["pos"] = torch.randint(0, npos, (t,), generator=gen, device=DEV, dtype=torch.int32)
    st["cos"], st["sin"] = _tables(npos, case["rot"])
    slots = torch.randperm(cap, generator=gen, device=DEV)[:t].to(torch.int32)
    if case["skip"]:  # padding tokens, which have no cache row
        slots[torch.rand(t, generator=gen, device=DEV) < 0.1] = -1
    st["slots"] = slots
    # what the cache held before
    st["kc"], st["ks"] = _random_cache(gen, cap * hkv, d)
    st["vc"], st["vs"] = _random_cache(gen, cap * hkv, d)
    return st


def _prepare_attn(case, gen):
    hq, hkv, d, page, dt = (case[i] for i in ("hq", "hkv", "d", "page", "dt"))
    q_lens, k_lens = _q_k_lengths(case)
    # pages in the order in which many streams took them
    need = [-(-n // page) for n in k_lens]
    total = max(1, sum(need))
    order = list(range(total))
    random.Random(case["lens"] + 1).shuffle(order)
    width = max(1, max(need))
    table = torch.full((case["nseq"], width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    st = {"table": table.to(DEV)}
    st["kc"], st["ks"] = _random_cache(gen, total * hkv * page, d)
    st["vc"], st["vs"] = _random_cache(gen, total * hkv * page, d)
    starts = [0]
    for n in q_lens:
        starts.append(starts[-1] + n)
    st["q"] = _normal(gen, (starts[-1], hq, d), dt)
    st["q_start"], st["k_len"] = _i32(starts), _i32(k_lens)
    st["q_lens"], st["k_lens"], st["starts"], st["pages"] = q_lens, k_lens, starts, total
    return st


# ---------------------------------------------------------------- the framework's calls

def _prepare_own(st):
    from ai_engine_amd import conv, mx4

    c = st["case"]
    dt = {"f32": conv.DType.F32, "f16": conv.DType.F16, "bf16": conv.DType.BF16}[c["dt"]]
    t = TORCH[c["dt"]]

    def empty(*shape, dtype=torch.uint8):
        return torch.empty(shape, dtype=dtype, device=DEV)

    if c["kind"] == "round":
        rows, k, kp = c["rows"], c["k"], _padded(c["k"])
        st["quant"] = mx4.Mx4QuantSpec(rows=rows, k=k, dt=dt)
        st["dequant"] = mx4.Mx4DequantSpec(rows=rows, k=k, dt=dt)
        st["codes"], st["scales"], st["y"] = empty(rows, kp // 2), empty(rows, _scale_bytes(k)), empty(rows, k, dtype=t)
    elif c["kind"] == "linear":
        m, k, n, kp = c["m"], c["k"], c["cout"], _padded(c["k"])
        st["quant"] = mx4.Mx4QuantSpec(rows=m, k=k, dt=dt)
        st["pw"] = mx4.Mx4PwSpec(m=m, k=k, cout=n, act=conv.Activation[c["act"].upper()], residual=c["residual"], dt=dt)
        st["codes"], st["scales"], st["y"] = empty(m, kp // 2), empty(m, _scale_bytes(k)), empty(m, n, dtype=t)
    elif c["kind"] == "append":
        st["append"] = mx4.Kv4AppendSpec(tokens=c["tokens"], hq=c["hq"], hkv=c["hkv"], d=c["d"], rot=c["rot"],
                                         pairs=c["pairs"], norm=False, dt=dt, positions=st["cos"].shape[0],
                                         page=c["page"], pages=c["cap"] // c["page"])
        st["dequant"] = mx4.Mx4DequantSpec(rows=c["cap"] * c["hkv"], k=c["d"], dt=dt, code_stride=c["d"] // 2,
                                           scale_stride=c["d"] // 32)
        st["q"] = empty(c["tokens"], c["hq"], c["d"], dtype=t)
        st["k"], st["v"] = (empty(c["cap"] * c["hkv"], c["d"], dtype=t) for _ in range(2))
    else:
        st["spec"] = mx4.Kv4AttnSpec(nseq=c["nseq"], tokens=st["starts"][-1], hq=c["hq"], hkv=c["hkv"], d=c["d"],
                                     page=c["page"], pages=st["pages"], table_width=st["table"].shape[1],
                                     causal=c["causal"], dt=dt, max_len=max(st["k_lens"]))
        st["out"] = empty(st["starts"][-1], c["hq"], c["d"], dtype=t)
        n = st["spec"].workspace_bytes()
        st["ws"] = empty(n // 4, dtype=torch.float32) if n else None


def _run_own(st):
    kind = st["case"]["kind"]
    if kind == "round":
        st["quant"].run(st["x"], st["codes"], st["scales"])
        return st["dequant"].run(st["codes"], st["scales"], st["y"])
    if kind == "linear":
        st["quant"].run(st["x"], st["codes"], st["scales"])
        return st["pw"].run(st["codes"], st["scales"], st["w_codes"], st["w_scales"], st["bias"], st["res"], st["y"])
    if kind == "append":
        st["append"].run(st["x"], None, None, st["cos"], st["sin"], st["pos"], st["slots"], st["q"], st["kc"], st["ks"],
                         st["vc"], st["vs"])
        st["dequant"].run(st["kc"], st["ks"], st["k"])
        st["dequant"].run(st["vc"], st["vs"], st["v"])
        return st["q"], st["k"], st["v"]
    return st["spec"].run(st["q"], st["kc"], st["ks"], st["vc"], st["vs"], st["q_start"], st["table"], st["k_len"],
                          st["out"], ws=st["ws"])


def run(state):
    if own:
        return _run_own(state)
    return {"round": _plain_round, "linear": _plain_linear, "append": _plain_append,
            "attn": _plain_attn}[state["case"]["kind"]](state)


# ---------------------------------------------------------------- the plain forms, fp32

def _plain_quant(x):
    """codes [rows, kp/2] and scales [rows, _scale_bytes(k)], kp the row's length in whole 128s."""
    rows, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, _padded(k) - k)).view(rows, -1, 32)
    codes, scales = _quant_blocks(x)
    return codes, torch.nn.functional.pad(scales, (0, _scale_bytes(k) - scales.shape[1]))


def _quant_blocks(x):
    """x [rows, blocks, 32] fp32."""
    m = x.abs().amax(-1, keepdim=True)
    # the exponent's bits less 2; of NaN and infinity all ones
    byte = ((m.view(torch.int32) >> 23) - 2).clamp(min=0)
    byte = torch.where(torch.isfinite(m), byte, 255)
    a = (x * ((254 - byte) << 23).view(torch.float32)).abs()
    mag = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = (mag + (torch.signbit(x).to(torch.uint8) << 3)).masked_fill(byte == 255, 0)
    codes = code[..., 0::2] | (code[..., 1::2] << 4)
    return codes.flatten(1).contiguous(), byte.flatten(1).to(torch.uint8)


def _values(codes, scales):
    """fp32 values [rows, blocks * 32] of codes [rows, blocks * 16] and scales [rows, blocks or more]."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    two = torch.stack([grid.repeat(16), grid.repeat_interleave(16)], -1)  # of a byte
    v = two[codes.int()].view(codes.shape[0], -1, 32)
    s = scales[:, :codes.shape[1] // 16].int()
    s = torch.where(s == 255, 0x7fc00000, torch.where(s == 0, 0x00400000, s << 23)).view(torch.float32)
    return (v * s[..., None]).view(codes.shape[0], -1)


def _plain_round(st):
    codes, scales = _plain_quant(st["x"])
    return _values(codes, scales)[:, :st["x"].shape[1]].to(st["x"].dtype)


def _act(v, act):
    if act == "relu":
        return torch.clamp(v, min=0)
    if act == "relu6":
        return torch.clamp(v, 0, 6)
    if act == "hardswish":
        return v * torch.clamp(v / 6 + 0.5, 0, 1)
    return v


def _plain_linear(st):
    a = _values(*_plain_quant(st["x"]))
    w = _values(st["w_codes"], st["w_scales"])
    y = _act(a @ w.t() + st["bias"].float(), st["case"]["act"])
    if st["res"] is not None:
        y = y + st["res"].float()
    return y.to(st["x"].dtype)


def _plain_append(st):
    c = st["case"]
    t, hq, hkv, d, rot, page, cap = (c[i] for i in ("tokens", "hq", "hkv", "d", "rot", "page", "cap"))
    x = st["x"].float()
    cos, sin = st["cos"][st["pos"].long()][:, None], st["sin"][st["pos"].long()][:, None]

    def rotate(y):
        if rot == 0:
            return y
        if c["pairs"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            z = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            z = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
        return torch.cat([z, y[..., rot:]], -1)

    q = rotate(x[:, :hq]).to(st["x"].dtype)
    slots = st["slots"].long()
    # heads' rows in the pages; the last one takes the tokens without a row
    row = (slots // page)[:, None] * (hkv * page) + torch.arange(hkv, device=DEV) * page + (slots % page)[:, None]
    row = torch.where(slots[:, None] < 0, cap * hkv, row).flatten()

    def put(new, codes, scales):
        c4, s4 = _quant_blocks(new.reshape(t * hkv, d // 32, 32))
        codes = torch.cat([codes, codes[:1]])
        scales = torch.cat([scales, scales[:1]])
        codes[row], scales[row] = c4, s4
        return _values(codes[:-1], scales[:-1]).to(st["x"].dtype)

    return q, put(rotate(x[:, hq:hq + hkv]), st["kc"], st["ks"]), put(x[:, hq + hkv:], st["vc"], st["vs"])


def _plain_attn(st):
    c = st["case"]
    n, hq, hkv, d, page = (c[i] for i in ("nseq", "hq", "hkv", "d", "page"))
    g, longest, rows = hq // hkv, max(1, max(st["k_lens"])), max(st["q_lens"])
    # every sequence's keys and values in order, padded to the longest
    j = torch.arange(longest, device=DEV)
    at = st["table"].long().clamp(min=0)[:, j // page] * (hkv * page) + j % page
    at = at[:, None] + torch.arange(hkv, device=DEV)[:, None] * page  # [n, hkv, longest]
    k = _values(st["kc"][at.flatten()], st["ks"][at.flatten()]).view(n * hkv, longest, d)
    v = _values(st["vc"][at.flatten()], st["vs"][at.flatten()]).view(n * hkv, longest, d)
    # the queries, padded likewise
    i = torch.arange(rows, device=DEV)
    lq, lk = st["q_start"][1:].long() - st["q_start"][:-1], st["k_len"].long()
    src = (st["q_start"][:-1].long()[:, None] + i).clamp(max=st["q"].shape[0] - 1)
    q = st["q"][src].float().view(n, rows, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(n * hkv, g * rows, d)
    s = torch.matmul(q * (1 / math.sqrt(d)), k.transpose(1, 2).contiguous()).view(n, hkv * g, rows, longest)
    hidden = j >= lk[:, None, None]
    if c["causal"]:
        hidden = hidden | (j > i[:, None] + (lk - lq)[:, None, None])
    s = s.masked_fill_(hidden[:, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp_(s.sub_(top))
    z = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n * hkv, g * rows, longest), v).view(n, hkv * g, rows, d)
    o = (o / torch.where(z == 0, 1.0, z)).permute(0, 2, 1, 3)
    return o[i < lq[:, None]].to(st["q"].dtype)


# ---------------------------------------------------------------- the definition, 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    return {"round": _exact_round, "linear": _exact_linear, "append": _exact_append,
            "attn": _exact_attn}[case["kind"]](st)


def _nearest(x):
    """The 4-bit values of x [rows, k] fp64, k in whole 32s, from the definition: a block's scale by its
    largest magnitude, each element the nearest value of the format, of two as near the one with the even code."""
    b = x.view(x.shape[0], -1, 32)
    big = b.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(big)  # big = f 2^e, f in [1/2, 1)
    e = torch.where(big == 0, torch.full_like(e, -127), (e - 3).clamp(min=-127))
    size = torch.ldexp(torch.ones_like(big), e)
    a = b.abs() / size
    # the spacing of the format at a: 1/2 below 2, 1 below 4, 2 above; round() takes the even multiple, which is the even code
    step = 0.5 + 0.5 * (a >= 2) + 1.0 * (a >= 4)
    v = (torch.round(a / step) * step).clamp(max=6)
    return (torch.copysign(v, b) * size).view(x.shape)


def _wide(x):
    k = x.shape[-1]
    return torch.nn.functional.pad(x.double(), (0, -k % 32))


def _exact_round(st):
    x = st["x"]
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for r in range(0, x.shape[0], 8192):
        out[r:r + 8192] = _nearest(_wide(x[r:r + 8192]))[:, :x.shape[1]]
    return out


def _decode(codes, scales):
    """The values of stored rows, fp64: sign, exponent and mantissa of each nibble."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    e, f = (c >> 1) & 3, (c & 1).double()
    mag = torch.where(e == 0, f / 2, torch.ldexp(1 + f / 2, e - 1))
    v = torch.where(c >= 8, -mag, mag)
    scales = scales[:, :codes.shape[1] // 16]
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.long() - 127)
    return v * s.repeat_interleave(32, -1)


def _exact_linear(st):
    c = st["case"]
    w = _decode(st["w_codes"], st["w_scales"])[:, :c["k"]]
    wt = w.t().contiguous()
    y = torch.empty(c["m"], c["cout"], dtype=torch.float64, device=DEV)
    for r in range(0, c["m"], 8192):
        a = _nearest(_wide(st["x"][r:r + 8192]))[:, :c["k"]].contiguous()
        v = a @ wt + st["bias"].double()
        if c["act"] in ("relu", "relu6"):
            v = v.clamp(min=0, max=6 if c["act"] == "relu6" else math.inf)
        elif c["act"] == "hardswish":
            v = v * ((v + 3).clamp(0, 6) / 6)
        if st["res"] is not None:
            v += st["res"][r:r + 8192].double()
        y[r:r + 8192] = v
    return y


def _exact_append(st):
    c = st["case"]
    t, hq, hkv, d, rot, page = (c[i] for i in ("tokens", "hq", "hkv", "d", "rot", "page"))
    x = st["x"].double()
    if rot:
        i = torch.arange(rot // 2, device=DEV)
        first, second = (2 * i, 2 * i + 1) if c["pairs"] else (i, i + rot // 2)
        turn = torch.complex(st["cos"].double(), st["sin"].double())[st["pos"].long()][:, None]
        z = torch.complex(x[:, :hq + hkv][..., first], x[:, :hq + hkv][..., second]) * turn
        x[:, :hq + hkv, first], x[:, :hq + hkv, second] = z.real, z.imag
    keep = torch.nonzero(st["slots"] >= 0).flatten()
    slot = st["slots"][keep].long()
    out = [x[:, :hq].contiguous()]
    for part, codes, scales in ((x[:, hq:hq + hkv], st["kc"], st["ks"]), (x[:, hq + hkv:], st["vc"], st["vs"])):
        # a key on the border between two 4-bit values after its rotation falls to one side in 64 bits and to the
        # other in 32; both are right, and there are few
        held = _decode(codes, scales).view(-1, hkv, page, d)
        for h in range(hkv):
            held[slot // page, h, slot % page] = _nearest(part[keep, h].contiguous())
        out.append(held.view(-1, d))
    return tuple(out)


def _exact_attn(st):
    c = st["case"]
    hq, hkv, d, page = (c[i] for i in ("hq", "hkv", "d", "page"))
    out = torch.zeros(st["starts"][-1], hq, d, dtype=torch.float64, device=DEV)
    kc, ks, vc, vs = (st[i].view(st["pages"], hkv, page, -1) for i in ("kc", "ks", "vc", "vs"))
    for b in range(c["nseq"]):
        lq, lk, q0 = st["q_lens"][b], st["k_lens"][b], st["starts"][b]
        if lq == 0 or lk == 0:
            continue
        pages = st["table"][b, :-(-lk // page)].long()
        for h in range(hkv):
            k = _decode(kc[pages, h].flatten(0, 1)[:lk], ks[pages, h].flatten(0, 1)[:lk])
            v = _decode(vc[pages, h].flatten(0, 1)[:lk], vs[pages, h].flatten(0, 1)[:lk])
            kt = k.t().contiguous()
            for qh in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                s = st["q"][q0:q0 + lq, qh].double() @ kt / math.sqrt(d)
                if c["causal"]:
                    seen = torch.arange(lq, device=DEV)[:, None] + (lk - lq)
                    s[torch.arange(lk, device=DEV)[None] > seen] = -math.inf
                lse = torch.logsumexp(s, -1, keepdim=True)
                p = torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse))
                out[q0:q0 + lq, qh] = p @ v
    return out
