"""A plain 64-bit implementation of the operators over paged caches, and the
bounds on how far the kernels may be from it."""
import math

import torch

PAGE = 32
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}


def half_step(dtype):
    """Largest relative error of a rounding to the type."""
    return torch.finfo(dtype).eps / 2


class Case:
    """Pools, table and activations of B sequences.  news / lens: new tokens
    and lengths with them; lead / tail: padding tokens around the chunks."""

    def __init__(self, news, lens, hq, hkv, d, io, kv, col=False, lead=0, tail=0, pad=0, seed=0, spare=3, gain=1.0,
                 device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed + 1)
        self.news, self.lens, self.hq, self.hkv, self.d, self.col = news, lens, hq, hkv, d, col
        self.io, self.kv, self.device = TYPES[io], TYPES[kv], device
        starts = [lead]
        for n in news:
            starts.append(starts[-1] + n)
        self.starts, self.n = starts, starts[-1] + tail
        need = [-(-n // PAGE) for n in lens]
        self.n_pages = sum(need) + spare
        order = torch.randperm(self.n_pages, device=device, generator=g).tolist()
        self.bps = max(max(need), 1)
        self.pages = [[order.pop() for _ in range(n)] for n in need]
        rows = [p + [2 ** 30 + i if i % 2 else -7 for i in range(self.bps - len(p))] for p in self.pages]
        self.table = torch.tensor(rows, dtype=torch.int32, device=device)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=device)
        # Pages of no sequence, and positions past a sequence's end, hold NaN.
        self.k, self.v = (torch.full((self.n_pages, hkv, d, PAGE), math.nan, device=device).to(self.kv) for _ in range(2))
        for b, n in enumerate(lens):
            for x in (self.k, self.v):
                full = torch.full((need[b] * PAGE, hkv, d), math.nan, device=device)
                full[:n] = torch.randn(n, hkv, d, device=device, generator=g) * (gain if x is self.k else 1.0)
                self._put(x, b, full)
        self.q, self.out = self.act(hq, pad, g, gain), self.act(hq, pad, None)

    def _put(self, pool, b, full):
        if not self.pages[b]:
            return
        blocks = full.reshape(-1, PAGE, self.hkv, self.d).permute(0, 2, 3, 1).contiguous().to(self.kv)
        bits = torch.uint8 if pool.element_size() == 1 else torch.int16
        pool.view(bits)[torch.tensor(self.pages[b], device=self.device)] = blocks.view(bits)

    def act(self, heads, pad=0, g=None, gain=1.0):
        """An activation tensor in the case's layout: random, or all 77."""
        rows = heads * self.d
        shape = (rows, self.n) if self.col else (self.n, rows)
        buf = torch.full((shape[0], shape[1] + pad), 77.0, device=self.device, dtype=self.io)
        if g is not None:
            buf[:, :shape[1]] = (torch.randn(*shape, device=self.device, generator=g) * gain).to(self.io)
        return buf[:, :shape[1]]

    def tokens(self, t):
        """[n, rows] in 64 bits."""
        return (t.t() if self.col else t).double()

    def dense(self, pool, b, length=None):
        """[length, hkv, d] in 64 bits: what the pages of sequence b hold."""
        length = self.lens[b] if length is None else length
        if length == 0:
            return torch.zeros(0, self.hkv, self.d, dtype=torch.float64, device=self.device)
        bits = torch.uint8 if pool.element_size() == 1 else torch.int16
        at = torch.tensor(self.pages[b], device=self.device)
        p = pool.view(bits)[at].view(pool.dtype).double().permute(0, 3, 1, 2)
        return p.reshape(-1, self.hkv, self.d)[:length]

    def batch(self, A, max_new=None, max_kv=None):
        return A.chunk_batch(self.k, self.v, self.table, self.q_start, self.kv_lens, self.n,
                             max_new or max(1, max(self.news)), max_kv or max(1, max(self.lens)), self.hkv, self.d)

    def layout(self, A):
        return A.HL_ACT_COLMAJOR if self.col else A.HL_ACT_TOKENMAJOR

    def run_attn(self, A, window=0, n_sink=0, scale=0.0, num_splits=0, **kw):
        a = A.attn_chunk_args(self.batch(A, **kw), self.q, self.out, self.hq, act_layout=self.layout(A), window=window,
                              n_sink=n_sink, scale=scale, num_splits=num_splits)
        ws = A.attn_chunk_workspace(a)
        A.attn_chunk(a, ws)
        return a, ws


def attn_reference(c, window=0, n_sink=0, scale=0.0, hidden_pages=()):
    """(out, bound) [n, hq*d] in 64 bits; NaN-free zeros where nothing is seen.
    The bound on |kernel - out|, with A = sum_j p_j |v_j| and u(t) the half step
    of a type:
      scores   products of d terms summed in fp32 in any order, of operands
               split to 2^-22 at worst (fp16 in two parts), scaled once and
               exponentiated: ds = (d + 16) 2^-24 + 2^-22 of scale sum |q k|,
               and 2^-22 of each weight; numerator and denominator: 4 ds A
      weights  rounded to the operand type once (u) or in two parts (u^2, fp16
               not below 2^-25 of the largest): that of A
      sums     len fp32 additions and the joins: (len + 64) 2^-24 A twice
      output   u(io) |out|"""
    scale = scale or 1.0 / math.sqrt(c.d)
    op = torch.float16 if c.kv == torch.float8_e4m3fn else c.kv
    high = c.io == torch.float32 or (c.io == torch.float16 and op == torch.bfloat16)
    u = half_step(op) ** 2 if high else half_step(op)
    out = torch.zeros(c.n, c.hq * c.d, dtype=torch.float64, device=c.device)
    bound = torch.zeros_like(out)
    q = c.tokens(c.q)
    grp = c.hq // c.hkv
    for b, (t, length) in enumerate(zip(c.news, c.lens)):
        if t == 0:
            continue
        k, v = c.dense(c.k, b), c.dense(c.v, b)
        i = torch.arange(length - t, length, device=c.device)[:, None]
        j = torch.arange(length, device=c.device)[None]
        seen = j <= i
        if window:
            seen = seen & ((i - j < window) | (j < n_sink))
        for blk in hidden_pages:
            seen = seen & (j // PAGE != blk)
        lo = c.starts[b]
        for h in range(c.hq):
            qh = q[lo:lo + t, h * c.d:(h + 1) * c.d]
            kh, vh = k[:, h // grp], v[:, h // grp]
            o, bd = torch.zeros(t, c.d, dtype=torch.float64, device=c.device), None
            bd = torch.zeros_like(o)
            if length:
                s = (qh @ kh.t().contiguous()) * scale
                s = torch.where(seen, s, -math.inf)
                top = s.amax(-1, keepdim=True)
                top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
                p = torch.exp(s - top)
                total = p.sum(-1, keepdim=True)
                p = torch.where(total > 0, p / total, torch.zeros_like(p))
                # a weight of exactly zero leaves its value out, whatever it is
                vz = [torch.where(torch.isfinite(vh), vh, torch.zeros_like(vh))]
                o = p @ vz[0]
                bad = ~torch.isfinite(vh)
                for jj in bad.any(-1).nonzero()[:, 0].tolist():
                    o = torch.where(seen[:, jj:jj + 1] & bad[jj], o + vh[jj], o)
                if torch.isfinite(k).all() and torch.isfinite(v).all():
                    mass = p @ vh.abs()
                    ds = ((c.d + 16) * 2.0 ** -24 + 2.0 ** -22) * scale * torch.where(
                        seen, qh.abs() @ kh.abs().t().contiguous(), torch.zeros_like(s)).amax(-1, keepdim=True)
                    low = 2.0 ** -25 * length * vh.abs().amax() if op == torch.float16 else 0.0
                    bd = mass * (torch.expm1(4 * ds) + 2.0 ** -21 + u + 2 * (length + 64) * 2.0 ** -24) + low
                    # below 2^-14 fp16 values are 2^-24 apart: off by 2^-25
                    bd = bd + (half_step(c.io) * o.abs() * 1.01).clamp_min(2.0 ** -25 if c.io == torch.float16 else 1e-37)
            out[lo:lo + t, h * c.d:(h + 1) * c.d] = o
            bound[lo:lo + t, h * c.d:(h + 1) * c.d] = bd
    return out, bound


def check_attn(c, **kw):
    ref, bound = attn_reference(c, **kw)
    got = c.tokens(c.out)
    inside = torch.zeros(c.n, dtype=torch.bool, device=c.device)
    for b, t in enumerate(c.news):
        inside[c.starts[b]:c.starts[b] + t] = True
    assert (got[~inside] == 77).all(), "tokens outside the chunks were written"
    off = (got - ref).abs()[inside] / bound[inside].clamp_min(1e-300)
    assert torch.isfinite(got[inside]).all(), "not finite"
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} times the bound, error {float((got - ref).abs()[inside].max()):.3g}"
    return worst
