"""An attention block over streams, as a hybrid network has it between its
convolution stages: the pointwise projection to queries, keys and values, head
norms and rotation into the cache, attention over the cache, the pointwise
projection back with the residual.

    y = x + W_out attention(norm, rotate(W_qkv x))

The two projections are the framework's 1x1 convs (ConvOp), the rest is
`attn`.  `step` takes the next tokens of every stream -- a whole frame or prompt
the first time, one token later -- and a context that all streams share can be
put in front once with `share`.

    block = AttnBlock(c=64, hq=4, hkv=2, d=32, streams=8, capacity=2048, weights=w, dt=DType.F16)
    y = block.step(frames)        # [8, tokens, 64]
    y = block.step(next_tokens)   # [8, 1, 64]

With `cache4` the cache holds keys and values in 4 bits (microscaled, in pages of
`page` rows; see `mx4`), a quarter of the 16-bit one's bytes, and one launch norms, rotates
and stores a step's rows.  With `proj4` the projections run in 4 bits as well: the
weights are quantised once, the rows on their way.
"""
from __future__ import annotations

from . import conv, mx4
from .attn import AttnSpec, QkNormRopeSpec
from .conv import AihError, ConvOp, DType


def rotation_tables(positions: int, rot: int, theta: float = 10000.0, device="cuda:0"):
    """(cosines, sines) [positions, rot/2] fp32 of the angles p theta^(-2i/rot)."""
    import torch

    half = rot // 2
    freq = theta ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return ang.cos().float().to(device), ang.sin().float().to(device)


class AttnBlock:
    """weights: w_qkv [(hq + 2 hkv) d, c], b_qkv, w_out [c, hq d], b_out, and the norms' wq, wk [d] (fp32
    arrays); capacity: cache rows of a stream; causal: a token sees the tokens up to its own (else the
    whole step's); prefix: rows kept for `share`; cache4, page: a 4-bit cache (d in whole 32s up to 256, rot in
    whole 16s, no prefix) in pages of so many rows (a power of two, 16 to 4096); proj4: 4-bit projections. Steps
    follow one another: on one stream, or with a wait in between.

    Besides the cache a block holds the buffers of its longest step: queries, results and the attention's workspace,
    (d + 2) fp32 values a token and query head for every part of the keys. That is large for whole prompts behind a
    shared context, whose keys are always in two parts or more (16 x 1024 tokens, 32 heads of 128: 545 MB)."""

    def __init__(self, c, hq, hkv, d, streams, capacity, weights, dt=DType.F32, rot=None, causal=True, prefix=0,
                 eps=1e-6, theta=10000.0, device="cuda:0", cache4=False, page=64, proj4=False):
        import numpy as np
        import torch

        if c % 8:
            raise AihError(f"c must be a multiple of 8, not {c}")
        self.c, self.hq, self.hkv, self.d, self.dt = c, hq, hkv, d, dt
        self.streams, self.capacity, self.causal, self.eps = streams, capacity, causal, eps
        self.rot, self.prefix, self.shared = d if rot is None else rot, prefix, 0
        self.device = device
        self._t = {DType.F32: torch.float32, DType.F16: torch.float16, DType.BF16: torch.bfloat16}[dt]

        def put(a):
            a = torch.from_numpy(a if a.dtype == np.float32 else a.view(np.int16)).to(device)
            return a if dt == DType.F32 else a.view(self._t)

        heads = hq + 2 * hkv
        for name, n in (("w_qkv", heads * d * c), ("b_qkv", heads * d), ("w_out", c * hq * d), ("b_out", c), ("wq", d),
                        ("wk", d)):
            if np.prod(np.shape(weights[name])) != n:  # what packs and reads them goes by the block's sizes alone
                raise AihError(f"{name} must hold {n} values, not {tuple(np.shape(weights[name]))}")
        self.cache4, self.proj4, self.page = cache4, proj4, page
        if cache4 and (prefix or d % 32 or not 32 <= d <= 256 or self.rot % 16):
            raise AihError("a 4-bit cache takes heads in whole 32s up to 256, rotations in whole 16s and no shared prefix")
        if cache4 and (type(page) is not int or not 16 <= page <= 4096 or page & (page - 1)):
            raise AihError(f"a 4-bit cache takes pages of a power of two rows, 16 to 4096, not {page!r}")
        if proj4:
            self.w_qkv = self._rows4(torch.as_tensor(weights["w_qkv"]).reshape(heads * d, c).float().to(device))
            self.w_out = self._rows4(torch.as_tensor(weights["w_out"]).reshape(c, hq * d).float().to(device))
        else:
            self.w_qkv = put(conv.pack_weights_conv(weights["w_qkv"], heads * d, c, 1, 1, 4, dt)[0])
            self.w_out = put(conv.pack_weights_conv(weights["w_out"], c, hq * d, 1, 1, 4, dt)[0])
        self.b_qkv = put(conv.pack_bias(weights["b_qkv"], heads * d, dt))
        self.b_out = put(conv.pack_bias(weights["b_out"], c, dt))
        self.wq, self.wk = (torch.as_tensor(weights[n]).to(device, self._t).contiguous() for n in ("wq", "wk"))
        self.cos, self.sin = rotation_tables(prefix + capacity, max(self.rot, 4), theta, device)
        if cache4:  # a stream's pages are its own, one after another
            per = -(-capacity // page)
            self.cache = mx4.kv4_cache(streams * per, page, hkv, d, device)
            self.table = torch.arange(streams * per, dtype=torch.int32, device=device).view(streams, per)
            self._first = torch.arange(streams, dtype=torch.int32, device=device) * (per * page)
        else:
            self.k = torch.zeros(streams * capacity, hkv, d, dtype=self._t, device=device)
            self.v = torch.zeros_like(self.k)
            self.pk = torch.zeros(max(prefix, 1), hkv, d, dtype=self._t, device=device)
            self.pv = torch.zeros_like(self.pk)
            self._first = torch.arange(streams, dtype=torch.int32, device=device) * capacity
        self._at = torch.arange(capacity, dtype=torch.int32, device=device)
        self._rows = torch.empty(2, 0, hq, d, dtype=self._t, device=device)  # queries and results of a step
        self._ws = torch.empty(0, dtype=torch.float32, device=device)
        self._plans = {}
        self.reset()

    def reset(self):
        """Forget every stream's tokens (what `share` holds stays)."""
        import torch

        self.length = 0
        self._len = torch.zeros(self.streams, dtype=torch.int32, device=self.device)

    def _check_rows(self, what, x, wanted, ok):
        """Refuse what the projection, which takes a bare address, would read as other rows or past their end."""
        at = self.cos.device
        if not ok or x.dtype != self._t or x.device != at or not x.is_contiguous():
            raise AihError(f"{what} takes a dense {wanted} {self._t} on {at}, not {tuple(x.shape)} "
                           f"{x.dtype} on {x.device}" + ("" if x.is_contiguous() else ", not dense"))

    def _rows4(self, x):
        """x [rows, k] in 4 bits: (codes, scales)."""
        import torch

        rows, k = x.shape
        dt = {torch.float32: DType.F32, torch.float16: DType.F16, torch.bfloat16: DType.BF16}[x.dtype]
        out = tuple(torch.empty(rows, n, dtype=torch.uint8, device=x.device)
                    for n in (mx4.code_bytes(k), mx4.scale_bytes(k)))
        return mx4.Mx4QuantSpec(rows=rows, k=k, dt=dt).run(x, *out)

    def _project(self, x, n, tokens):
        import torch

        heads = self.hq + 2 * self.hkv
        qkv = torch.empty(n * tokens, heads, self.d, dtype=self._t, device=self.device)
        if self.proj4:
            spec = mx4.Mx4PwSpec(m=n * tokens, k=self.c, cout=heads * self.d, dt=self.dt)
            return spec.run(*self._rows4(x.view(n * tokens, self.c)), *self.w_qkv, self.b_qkv, None, qkv)
        ConvOp(ih=tokens, iw=1, cin=self.c, cout=heads * self.d, dt=self.dt, n=n).run(
            x, self.w_qkv, self.b_qkv, None, qkv)
        return qkv

    def _norm_spec(self, tokens, rows):
        return QkNormRopeSpec(tokens=tokens, hq=self.hq, hkv=self.hkv, d=self.d, rot=self.rot, eps=self.eps,
                              dt=self.dt, positions=self.cos.shape[0], rows=rows)

    def share(self, x):
        """x [tokens, c] in the block's type, on the device: the context in front of every stream, read once for
        all by each step; no tokens: none any more."""
        import torch

        self._check_rows("share", x, f"[tokens, {self.c}]", x.dim() == 2 and x.shape[1] == self.c)
        tokens = x.shape[0]
        if tokens > self.prefix:
            raise AihError(f"{tokens} shared tokens, room for {self.prefix}")
        if self.length:
            raise AihError("share comes before the streams' tokens: their positions start behind it")
        if tokens:
            qkv = self._project(x, 1, tokens)
            q = torch.empty(tokens, self.hq, self.d, dtype=self._t, device=self.device)
            self._norm_spec(tokens, tokens).run(qkv, self.wq, self.wk, self.cos, self.sin, None, None, q, self.pk,
                                                self.pv)
        self.shared = tokens
        self._plans.clear()

    def _outgrown(self, buffer):
        """`buffer` is let go: by the plans, and only after the last step on the current stream."""
        import torch

        self._plans.clear()
        if buffer.is_cuda and buffer.numel():
            buffer.record_stream(torch.cuda.current_stream(buffer.device))

    def _plan(self, tokens):
        """The specs of a step of `tokens` tokens a stream, made once, and its part of the buffers, which all lengths
        share: the steps of a block follow one another on a stream."""
        import torch

        p = self._plans.get(tokens)
        if p is None:
            n = self.streams * tokens
            if self.cache4:
                pages, width = self.table.numel(), self.table.shape[1]
                spec = mx4.Kv4AttnSpec(nseq=self.streams, tokens=n, hq=self.hq, hkv=self.hkv, d=self.d, page=self.page,
                                       pages=pages, table_width=width, causal=self.causal, dt=self.dt,
                                       max_len=self.capacity)
                norm = mx4.Kv4AppendSpec(tokens=n, hq=self.hq, hkv=self.hkv, d=self.d, page=self.page, pages=pages,
                                         rot=self.rot, norm=True, eps=self.eps, dt=self.dt,
                                         positions=self.cos.shape[0])
            else:
                spec = AttnSpec(nseq=self.streams, tokens=n, rows=self.streams * self.capacity, hq=self.hq,
                                hkv=self.hkv, d=self.d, causal=self.causal, dt=self.dt, max_len=self.capacity,
                                prefix=self.shared)
                norm = self._norm_spec(n, self.streams * self.capacity)
            if self.proj4:
                out = mx4.Mx4PwSpec(m=n, k=self.hq * self.d, cout=self.c, residual=True, dt=self.dt)
            else:
                out = ConvOp(ih=tokens, iw=1, cin=self.hq * self.d, cout=self.c, residual=True, dt=self.dt,
                             n=self.streams)
            ws = spec.workspace_bytes()
            if n > self._rows.shape[1]:
                self._outgrown(self._rows)
                self._rows = torch.empty(2, n, self.hq, self.d, dtype=self._t, device=self.device)
            if ws // 4 > self._ws.shape[0]:
                self._outgrown(self._ws)
                self._ws = torch.empty(ws // 4, dtype=torch.float32, device=self.device)
            p = self._plans[tokens] = dict(
                norm=norm, attn=spec, out=out,
                q=self._rows[0, :n], o=self._rows[1, :n], ws=self._ws if ws else None, at=self._at[:tokens],
                q_start=torch.arange(0, n + 1, tokens, dtype=torch.int32, device=self.device))
        return p

    def step(self, x):
        """x [streams, tokens, c] in the block's type, on the device: the next tokens of every stream; returns
        [streams, tokens, c]."""
        import torch

        self._check_rows("step", x, f"[{self.streams}, tokens, {self.c}]",
                         x.dim() == 3 and x.shape[0] == self.streams and x.shape[2] == self.c)
        streams, tokens, _ = x.shape
        if tokens == 0:
            return torch.empty_like(x)
        if self.length + tokens > self.capacity:
            raise AihError(f"{self.length} + {tokens} tokens, room for {self.capacity} a stream")
        p = self._plan(tokens)
        at = self._len[:, None] + p["at"]
        pos, slots = (at + self.shared).flatten(), (at + self._first[:, None]).flatten()
        filled = self._len + tokens

        qkv = self._project(x, streams, tokens)
        if self.cache4:
            p["norm"].run(qkv, self.wq, self.wk, self.cos, self.sin, pos, slots, p["q"], *self.cache)
            p["attn"].run(p["q"], *self.cache, p["q_start"], self.table, filled, p["o"], ws=p["ws"])
        else:
            p["norm"].run(qkv, self.wq, self.wk, self.cos, self.sin, pos, slots, p["q"], self.k, self.v)
            p["attn"].run(p["q"], self.k, self.v, p["q_start"], self._first, filled, p["o"], prefix_k=self.pk,
                          prefix_v=self.pv, ws=p["ws"])
        y = torch.empty_like(x)
        if self.proj4:
            p["out"].run(*self._rows4(p["o"].view(streams * tokens, -1)), *self.w_out, self.b_out, x, y)
        else:
            p["out"].run(p["o"], self.w_out, self.b_out, x, y)
        self._len, self.length = filled, self.length + tokens
        return y
