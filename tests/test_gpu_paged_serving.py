"""GPU: the operators over paged caches together, as a server uses them.

Sequences get their prompts in chunks, one forks (sharing pages, copying the
part-filled one on write), all step token by token in ragged batches, a window
gives pages back, the pool is compacted; every output is compared with the
plain 64-bit attention over the sequence's whole history of rotated keys."""
import math

import pytest
import torch

from paged_util import PAGE, half_step

pytestmark = pytest.mark.gpu
HQ, HKV, D, BASE = 16, 4, 64, 1e4


class Server:
    def __init__(self, A, kv, io, n_pages=120, bps=24, layers=2, window=0, sinks=0):
        self.A, self.io, self.window, self.sinks, self.bps = A, io, window, sinks, bps
        self.pages = A.PagePool(n_pages)
        self.pools = [torch.full((n_pages, HKV, D, PAGE), math.nan, device="cuda").to(kv) for _ in range(2 * layers)]
        self.args = A.kv_pages_args(self.pools)
        self.layers, self.seqs = layers, []
        self.freqs = A.rope_freqs(D, BASE, A.rope_scaling(A.HL_ROPE_SCALE_YARN, 4.0, 512.0))
        self.ws = None
        self.kv = kv

    def add(self):
        self.seqs.append({"table": torch.full((self.bps,), -1, dtype=torch.int32), "len": 0,
                          "hist": [[] for _ in range(self.layers)]})
        return self.seqs[-1]

    def fork(self, s, length):
        t = self.add()
        self.pages.fork(s["table"], t["table"], length)
        t["len"] = length
        t["hist"] = [h[:length] for h in s["hist"]]
        return t

    def step(self, seqs, news, g):
        """One forward's attention parts in each layer; outputs checked."""
        A, n = self.A, sum(news)
        moves = [m for s, t in zip(seqs, news) if (m := self.pages.extend(s["table"], s["len"], s["len"] + t))]
        if moves:
            A.kv_pages_copy(self.args, torch.tensor(moves, dtype=torch.int32))
        for s, t in zip(seqs, news):
            s["len"] += t
        starts = [0]
        for t in news:
            starts.append(starts[-1] + t)
        table = torch.stack([s["table"] for s in seqs]).cuda()
        lists = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, [s["len"] for s in seqs])]
        for layer in range(self.layers):
            k_pool, v_pool = self.pools[2 * layer], self.pools[2 * layer + 1]
            b = A.chunk_batch(k_pool, v_pool, table, *lists, n, max(news), max(s["len"] for s in seqs), HKV, D)
            q, k, v = (torch.randn(n, h * D, device="cuda", generator=g).to(self.io) for h in (HQ, HKV, HKV))
            plain = (q.double(), k.double(), v.double())
            A.rope_store_chunk(A.rope_store_chunk_args(b, q, k, v, q, HQ, BASE, act_layout=A.HL_ACT_TOKENMAJOR,
                                                       freqs=self.freqs))
            out = torch.full_like(q, 77)
            a = A.attn_chunk_args(b, q, out, HQ, act_layout=A.HL_ACT_TOKENMAJOR, window=self.window, n_sink=self.sinks)
            need = A.attn_chunk_workspace_bytes(a)
            if self.ws is None or self.ws.numel() < need:
                self.ws = A.attn_chunk_workspace(a)
            A.attn_chunk(a, self.ws)
            self.check(layer, seqs, news, starts, plain, out.double())

    def check(self, layer, seqs, news, starts, plain, out):
        f = torch.tensor([float(h) + float(lo) for h, lo in zip(self.freqs.turns_hi[:D // 2], self.freqs.turns_lo[:D // 2])],
                         dtype=torch.float64, device="cuda")

        def spun(x, pos, heads):
            x = x.reshape(-1, heads, D)
            ang = (pos[:, None] * f * 2 * math.pi)[:, None]
            a, c = x[..., :D // 2], x[..., D // 2:]
            co, si = torch.cos(ang) * self.freqs.gain, torch.sin(ang) * self.freqs.gain
            return torch.cat([a * co - c * si, a * si + c * co], -1)

        for s, t, lo in zip(seqs, news, starts):
            pos = torch.arange(s["len"] - t, s["len"], device="cuda", dtype=torch.float64)
            # the history is what was written, rounded to the caches' type
            kr = spun(plain[1][lo:lo + t], pos, HKV).float().to(self.kv).double()
            vr = plain[2][lo:lo + t].reshape(-1, HKV, D).float().to(self.kv).double()
            s["hist"][layer] += list(zip(kr, vr))
            k = torch.stack([x[0] for x in s["hist"][layer]]).repeat_interleave(HQ // HKV, 1)
            v = torch.stack([x[1] for x in s["hist"][layer]]).repeat_interleave(HQ // HKV, 1)
            q = spun(plain[0][lo:lo + t], pos, HQ).float().to(self.io).double()
            z = torch.matmul(q.transpose(0, 1).contiguous(), k.permute(1, 2, 0).contiguous()) / math.sqrt(D)
            j = torch.arange(s["len"], device="cuda")
            i = pos.long()[:, None]
            seen = j <= i
            if self.window:
                seen = seen & ((i - j < self.window) | (j < self.sinks))
            p = torch.softmax(torch.where(seen, z, -math.inf), -1)
            want = torch.matmul(p, v.transpose(0, 1).contiguous()).transpose(0, 1).reshape(t, HQ * D)
            got = out[lo:lo + t]
            # Weights and outputs rounded once each; a key or query component
            # rounded the other way moves a score by half a step of its product
            # in one of 64 dims: 8 half steps cover the few that do.
            u = max(half_step(self.io), half_step(self.kv) if self.kv != torch.float8_e4m3fn else 0.0)
            lim = (8 * u + 2e-5) * torch.matmul(p, v.abs().transpose(0, 1).contiguous()).transpose(0, 1).reshape(t, HQ * D)
            if self.kv == torch.float8_e4m3fn:  # a flipped key component: 2^-4 of it
                lim = lim * 4 + 0.02
            assert torch.isfinite(got).all()
            assert ((got - want).abs() <= lim + 1e-6).all(), float(((got - want).abs() / (lim + 1e-6)).max())


@pytest.mark.parametrize("kv,io,window", [("bf16", "bf16", 0), ("f16", "f32", 0), ("fp8", "bf16", 0), ("bf16", "f32", 96)])
def test_serving(hl, kv, io, window):
    from hippo_leap_amd import attention as A
    from paged_util import TYPES
    g = torch.Generator(device="cuda").manual_seed(3)
    sv = Server(A, TYPES[kv], TYPES[io], window=window, sinks=3 if window else 0)
    a, b, c = sv.add(), sv.add(), sv.add()
    print("prompts in chunks", flush=True)
    sv.step([a, b], [130, 45], g)
    sv.step([a, c], [77, 1], g)
    print("mixed", flush=True)
    sv.step([a, b, c], [1, 33, 260], g)
    print("fork", flush=True)
    d = sv.fork(a, a["len"])
    e = sv.fork(a, 100)  # from an earlier point
    for i in range(4):
        sv.step([a, b, c, d, e], [1, 1, 1, 1, 1], g)
    print("verify", flush=True)
    sv.step([a, d, e], [5, 3, 40], g)
    print("release", flush=True)
    sv.pages.release(b["table"])
    sv.seqs = [s for s in sv.seqs if s is not b]
    if window:
        for s in sv.seqs:
            first = max(1, (s["len"] - window + 1) // PAGE)
            sv.pages.release(s["table"], 1, first - 1)
    print("compact", flush=True)
    tables = torch.stack([s["table"] for s in sv.seqs])
    moves = sv.pages.compact(tables)
    assert len(moves)
    A.kv_pages_copy(sv.args, moves)
    for s, row in zip(sv.seqs, tables):
        s["table"].copy_(row)
    # what lies above the pages in use is no one's: poison it
    used = max(int(t.max()) for t in tables) + 1
    for p in sv.pools:
        p[used:] = torch.full((1,), math.nan, device="cuda").to(p.dtype) if p.element_size() > 1 else p[used:]
    print("after", flush=True)
    f = sv.add()
    sv.step([a, c, d, e, f], [1, 1, 2, 1, 50], g)


@pytest.mark.parametrize("kv", ["f16", "bf16", "fp8"])
def test_agrees_with_the_decode_step(hl, kv):
    """The same new token through the two chunk calls and through the
    framework's fused decode step over the same pages (no scaling: the step
    has none), short positions so that both angles agree."""
    from hippo_leap_amd import attention as A
    from paged_util import Case
    B, L = 3, 65
    c = Case([1] * B, [L, L - 31, L - 64], 8, 2, 128, "f32", kv)
    g = torch.Generator(device="cuda").manual_seed(8)
    q, k, v = (torch.randn(B, h * 128, device="cuda", generator=g) for h in (8, 2, 2))
    out = torch.empty(B, 8 * 128, device="cuda")
    table = c.table.clamp(0, c.n_pages - 1)
    pools = [c.k.clone(), c.v.clone()]
    positions = c.kv_lens - 1
    M = 32 * c.bps
    rs = A.rope_store_args(q.clone(), k.clone(), v, *pools, 8, 2, 128, M, int(positions.max()), 1e4, positions=positions,
                           kv_layout=A.HL_KV_PAGED32, block_table=table)
    at = A.decode_args(rs._tensors[0], *pools, out, 8, 2, 128, M, L, kv_layout=A.HL_KV_PAGED32, block_table=table)
    A.decode_step(rs, at, A.decode_step_workspace(rs, at))
    q2, out2 = torch.empty_like(q), torch.empty_like(out)
    b = A.chunk_batch(c.k, c.v, c.table, c.q_start, c.kv_lens, B, 1, L, 2, 128)
    A.rope_store_chunk(A.rope_store_chunk_args(b, q, k, v, q2, 8, 1e4, act_layout=A.HL_ACT_TOKENMAJOR))
    a = A.attn_chunk_args(b, q2, out2, 8, act_layout=A.HL_ACT_TOKENMAJOR)
    A.attn_chunk(a, A.attn_chunk_workspace(a))
    torch.cuda.synchronize()
    # one rounding of a key component may fall the other way
    assert (out - out2).abs().max() <= (2e-2 if kv == "fp8" else 2e-3) * out.abs().max()
    for x, y in zip(pools, (c.k, c.v)):
        for s in range(B):
            d = (c.dense(x, s) - c.dense(y, s)).abs()
            assert d.max() <= 2 ** -4 * 4 if kv == "fp8" else d.max() <= 2 ** -8 * 4
            assert (d > 0).float().mean() < 0.01
