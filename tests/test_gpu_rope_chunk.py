"""GPU: hl_rope_store_chunk against the formulas in 64 bits."""
import math

import pytest
import torch

from paged_util import PAGE, Case, half_step

pytestmark = pytest.mark.gpu

# news, lens, hq, hkv, d, io, kv, rope_dim, pairs, scaling, norm, col
CASES = {
    "one": ([1], [1], 4, 4, 64, "f32", "f16", 64, "half", "none", False, False),
    "decode": ([1] * 5, [1, 32, 33, 5000, 40000], 32, 8, 128, "bf16", "bf16", 128, "half", "llama3", False, False),
    "decode_col": ([1] * 3, [100, 31, 64], 32, 8, 64, "f32", "fp8", 32, "inter", "yarn", True, True),
    "prompt": ([100], [100], 8, 2, 64, "f16", "f16", 64, "half", "linear", False, False),
    "chunk": ([70], [1000], 16, 4, 128, "bf16", "bf16", 128, "inter", "yarn", True, False),
    "chunk_col": ([65, 3], [97, 200], 8, 2, 128, "f32", "bf16", 64, "half", "none", True, True),
    "ragged": ([0, 33, 1, 200, 2], [50, 33, 77, 333, 66], 28, 4, 64, "bf16", "fp8", 64, "half", "llama3", True, False),
    "no_rotation": ([40], [50], 8, 2, 64, "f32", "f16", 0, "half", "none", True, False),
    "many_heads": ([300], [400], 64, 8, 128, "f16", "f16", 126, "inter", "none", False, False),
}
SCALE = {"none": {}, "linear": {"factor": 4.0}, "llama3": {"factor": 8.0, "original_len": 8192.0},
         "yarn": {"factor": 4.0, "original_len": 4096.0}}


def frequencies(scaling, r, base):
    """The rotation per position of each pair, from the formulas, and the gain."""
    out = []
    gain = 1.0
    f = SCALE[scaling].get("factor", 1.0)
    n = SCALE[scaling].get("original_len", 0.0)
    for i in range(r // 2):
        w = base ** (-2.0 * i / r)
        if scaling == "linear":
            w /= f
        elif scaling == "llama3":
            turns = n * w / (2 * math.pi)
            if turns <= 1:
                w /= f
            elif turns < 4:
                w = w * (turns - 1) / 3 + w / f * (4 - turns) / 3
        elif scaling == "yarn":
            at = [math.log(n / (t * 2 * math.pi)) / math.log(base) * r / 2 for t in (32, 1)]
            lo, hi = max(0, math.floor(at[0])), min(r - 1, math.ceil(at[1]))
            part = 0.0 if i <= lo else 1.0 if i >= hi else (i - lo) / (hi - lo)
            w = w * (1 - part) + w / f * part
            gain = 0.1 * math.log(f) + 1
        out.append(w)
    return torch.tensor(out, dtype=torch.float64), gain


def kind_of(A, scaling):
    return {"none": A.HL_ROPE_SCALE_NONE, "linear": A.HL_ROPE_SCALE_LINEAR, "llama3": A.HL_ROPE_SCALE_LLAMA3,
            "yarn": A.HL_ROPE_SCALE_YARN}[scaling]


def reference(c, x, heads, w, r, pairs, scaling, base, eps):
    """[n, heads, d] in 64 bits and the bound on its fp32 value: the rotation's
    angle is off by 2^-23 of a turn and cos and sin by 2^-22, the norm by
    (d + 8) 2^-24, each product and sum by 2^-24."""
    x = c.tokens(x).reshape(c.n, heads, c.d).clone()
    size = torch.zeros(c.n, heads, 1, dtype=torch.float64, device="cuda")
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        size = size + (c.d + 8) * 2.0 ** -24
    bound = x.abs() * size
    freq, gain = frequencies(scaling, r, base) if r else (torch.zeros(0, dtype=torch.float64), 1.0)
    pos = torch.zeros(c.n, dtype=torch.float64)
    for b, t in enumerate(c.news):
        pos[c.starts[b]:c.starts[b] + t] = torch.arange(c.lens[b] - t, c.lens[b], dtype=torch.float64)
    ang = (pos[:, None] * freq).cuda()[:, None]
    co, si = torch.cos(ang) * gain, torch.sin(ang) * gain
    i0, i1 = (slice(0, r // 2), slice(r // 2, r)) if pairs == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, e = x[..., i0].clone(), x[..., i1].clone()
    x[..., i0], x[..., i1] = a * co - e * si, a * si + e * co
    mag = (a.abs() + e.abs()) * gain * (2 * math.pi * 2.0 ** -23 + 2.0 ** -22 + 4 * 2.0 ** -24 + size)
    bound[..., i0], bound[..., i1] = mag, mag
    return x, bound + 1e-37


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_matches_formulas(hl, name, in_place):
    from hippo_leap_amd import attention as A
    news, lens, hq, hkv, d, io, kv, r, pairs, scaling, norm, col = CASES[name]
    print(f"rope {name} in_place {in_place}", flush=True)
    base, eps = 5e5, 1e-6
    c = Case(news, lens, hq, hkv, d, io, kv, col, lead=1, tail=2, pad=3, seed=len(name))
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = c.act(hkv, 3, g), c.act(hkv, 3, g)
    wq, wk = ((0.5 + torch.rand(d, device="cuda", generator=g)) for _ in range(2)) if norm else (None, None)
    q_ref, q_bound = reference(c, c.q, hq, wq, r, pairs, scaling, base, eps)
    k_ref, k_bound = reference(c, k, hkv, wk, r, pairs, scaling, base, eps)
    v_ref = c.tokens(v).reshape(c.n, hkv, d)
    q_in = c.tokens(c.q).clone()
    old = [c.k.clone(), c.v.clone()]
    freqs = A.rope_freqs(r, base, A.rope_scaling(kind_of(A, scaling), **SCALE[scaling])) if r else A.RopeFreqs()
    a = A.rope_store_chunk_args(c.batch(A), c.q, k, v, c.q if in_place else c.out, hq, base,
                                rope_style=A.HL_ROPE_HALF_SPLIT if pairs == "half" else A.HL_ROPE_INTERLEAVED,
                                q_norm_w=wq, k_norm_w=wk, eps=eps, act_layout=c.layout(A), freqs=freqs)
    A.rope_store_chunk(a)
    torch.cuda.synchronize()
    got = c.tokens(c.q if in_place else c.out)
    inside = torch.zeros(c.n, dtype=torch.bool, device="cuda")
    for b, t in enumerate(news):
        inside[c.starts[b]:c.starts[b] + t] = True
    assert torch.equal(got[~inside], q_in[~inside] if in_place else torch.full_like(q_in[~inside], 77))
    # below 2^-14 fp16 values are 2^-24 apart: a rounding there is off by 2^-25
    low = 2.0 ** -25 if io == "f16" else 0.0
    off = (got.reshape(c.n, hq, d) - q_ref).abs() - (half_step(c.io) * 1.01 * q_ref.abs()).clamp_min(low) - q_bound * 1.01
    worst = float(off[inside].max())
    assert worst <= 0, worst
    bits = torch.uint8 if kv == "fp8" else torch.int16
    for pool, before, ref, bound in ((c.k, old[0], k_ref, k_bound), (c.v, old[1], v_ref, torch.zeros_like(v_ref))):
        untouched = torch.ones(pool.shape[0], PAGE, dtype=torch.bool, device="cuda")
        for b, (t, n) in enumerate(zip(news, lens)):
            if not t:
                continue
            for p in range(n - t, n):
                untouched[c.pages[b][p // PAGE], p % PAGE] = False
            want = ref[c.starts[b]:c.starts[b] + t]
            have = c.dense(pool, b)[n - t:]
            lim = half_step(c.kv) * 1.01 * want.abs() + bound[c.starts[b]:c.starts[b] + t] * 1.1
            if kv == "fp8":  # subnormals step by 2^-9
                lim = lim.clamp_min(2.0 ** -10)
            if kv == "f16":
                lim = lim.clamp_min(2.0 ** -25)
            worst = float(((have - want).abs() - lim).max())
            assert worst <= 0, worst
        same = pool.view(bits).permute(0, 3, 1, 2)[untouched] == before.view(bits).permute(0, 3, 1, 2)[untouched]
        assert same.all(), "a position of no new token was written"


def test_fp8_saturates_and_keeps_nan(hl):
    from hippo_leap_amd import attention as A
    c = Case([4], [40], 4, 2, 64, "f32", "fp8")
    k, v = c.act(2), c.act(2)
    k[:], v[:] = 0.0, 0.0
    v[0, 0], v[0, 1], v[0, 2], v[0, 3] = 1e6, -math.inf, math.nan, 447.0
    A.rope_store_chunk(A.rope_store_chunk_args(c.batch(A), c.q, k, v, c.out, 4, 1e4, act_layout=c.layout(A)))
    have = c.dense(c.v, 0)[36, 0]
    assert have[0] == 448 and have[1] == -448 and torch.isnan(have[2]) and have[3] == 448


def test_fused_projection_views(hl):
    """q, k and v as slices of one fused projection's rows, rotated in place."""
    from hippo_leap_amd import attention as A
    c = Case([50, 1], [90, 33], 8, 2, 64, "bf16", "bf16")
    g = torch.Generator(device="cuda").manual_seed(4)
    fused = torch.randn(c.n, 12 * 64, device="cuda", generator=g).to(torch.bfloat16)
    parts = [fused[:, :512], fused[:, 512:640], fused[:, 640:]]
    apart = [p.clone() for p in parts]
    out = torch.empty_like(apart[0])
    A.rope_store_chunk(A.rope_store_chunk_args(c.batch(A), *apart, out, 8, 1e4, act_layout=c.layout(A)))
    want = (out, c.k.clone(), c.v.clone())
    A.rope_store_chunk(A.rope_store_chunk_args(c.batch(A), *parts, parts[0], 8, 1e4, act_layout=c.layout(A)))
    assert torch.equal(parts[0], want[0])
    assert torch.equal(c.k.view(torch.int16), want[1].view(torch.int16))
    assert torch.equal(c.v.view(torch.int16), want[2].view(torch.int16))
    assert torch.equal(parts[1], apart[1]) and torch.equal(parts[2], apart[2])


def test_missing_pages_are_not_stored(hl):
    """Tokens whose page is not in the pool, or whose position lies below
    zero: q is rotated, nothing is stored."""
    from hippo_leap_amd import attention as A
    c = Case([70], [100], 4, 2, 64, "f32", "f16")
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = c.act(2, 0, g), c.act(2, 0, g)
    c.table[0, 2] = c.n_pages + 5
    before = [p.view(torch.int16)[c.pages[0][2]].clone() for p in (c.k, c.v)]
    A.rope_store_chunk(A.rope_store_chunk_args(c.batch(A), c.q, k, v, c.out, 4, 1e4, act_layout=c.layout(A)))
    for p, old in zip((c.k, c.v), before):
        assert torch.equal(p.view(torch.int16)[c.pages[0][2]], old)
    assert torch.isfinite(c.out).all()
    c.kv_lens.fill_(30)  # 40 tokens at positions -40 .. -1
    A.rope_store_chunk(A.rope_store_chunk_args(c.batch(A), c.q, k, v, c.out, 4, 1e4, act_layout=c.layout(A)))
    c.lens = [30]
    assert (c.dense(c.v, 0) - c.tokens(v)[40:].reshape(30, 2, 64)).abs().max() < 2 ** -8


def test_captured_store_reads_its_lists(hl):
    from hippo_leap_amd import attention as A
    c = Case([3, 3], [40, 70], 4, 2, 64, "f32", "f16")
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = c.act(2, 0, g), c.act(2, 0, g)
    a = A.rope_store_chunk_args(c.batch(A), c.q, k, v, c.out, 4, 1e4, act_layout=c.layout(A))
    A.rope_store_chunk(a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.rope_store_chunk(a)
    for lens in ([40, 70], [12, 33], [3, 64]):
        c.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = (c.out.clone(), c.k.clone(), c.v.clone())
        A.rope_store_chunk(a)
        torch.cuda.synchronize()
        assert torch.equal(got[0], c.out)
        for b in range(2):
            for x, y in zip(got[1:], (c.k, c.v)):
                assert torch.equal(c.dense(x, b, lens[b]), c.dense(y, b, lens[b]))
            want = c.tokens(v)[3 * b:3 * b + 3].reshape(3, 2, 64)
            assert (c.dense(c.v, b, lens[b])[-3:] - want).abs().max() < 2 ** -8
