"""The operators of serving over a paged cache, as a serving program calls them:
the plain form of each in elementary torch operations, and the framework's own
(`own` true) on the same inputs.

  attn   attn_chunk: attention of the new tokens of B sequences (a prompt's
         next chunk, proposed tokens to verify, single tokens, or a mixture)
         over HL_KV_PAGED32 caches, with a sliding window and first tokens
         that stay visible where the model has them
  rope   rope_store_chunk: qkNorm, rotary positions and the store of the new
         tokens' k and v into the pages
  copy   kv_pages_copy: pages of every layer's K and V pool copied to others
         (a forked sequence's last page, a compacted pool)

Sizes are those of the benchmark's and tests' shapes (TinyLlama, Llama-3.2-1B,
Llama-3-8B, Qwen3-30B-A3B attention) and of generic ones between them.
"""
import math

import numpy as np
import torch

own = False

PAGE = 32
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "fp8": 1}
EPS = 1e-6


def listed():
    return [
        # The smallest attention call: one token of a Llama-3.2-1B-shaped
        # model whose window has begun to slide, fp32 activations.
        {"name": "attn_one_f16_window", "kind": "attn", "b": 1, "new": 1, "len": 1500, "ragged": False, "hq": 32,
         "hkv": 8, "d": 64, "io": "f32", "kv": "f16", "window": 1024, "sinks": 4, "col": False},
        # A serving batch deep in long contexts, Qwen3-30B-A3B attention: the
        # window and the sinks are all that is read of 32K positions.
        {"name": "attn_b16_32k_window", "kind": "attn", "b": 16, "new": 1, "len": 32769, "ragged": True, "hq": 32,
         "hkv": 4, "d": 128, "io": "f32", "kv": "bf16", "window": 4096, "sinks": 4, "col": False},
        # Five proposed tokens for each of eight sequences, verified at once,
        # Llama-3-8B attention.
        {"name": "attn_verify_b8", "kind": "attn", "b": 8, "new": 5, "len": 2049, "ragged": True, "hq": 32, "hkv": 8,
         "d": 128, "io": "bf16", "kv": "bf16", "window": 0, "sinks": 0, "col": False},
        # The last 512 tokens of an 8K prompt taken in chunks, Llama-3-8B.
        {"name": "attn_chunk512_8k", "kind": "attn", "b": 1, "new": 512, "len": 8192, "ragged": False, "hq": 32,
         "hkv": 8, "d": 128, "io": "bf16", "kv": "bf16", "window": 0, "sinks": 0, "col": False},
        # A step of continuous batching: most sequences add one token, every
        # eighth brings a chunk of its prompt; Llama-3.2-1B attention.
        {"name": "attn_mixed_b26", "kind": "attn", "b": 26, "new": 351, "len": 3001, "ragged": True, "hq": 32,
         "hkv": 8, "d": 64, "io": "f16", "kv": "f16", "window": 0, "sinks": 0, "col": False},
        # A long prompt's chunk over an fp8 cache, Qwen3-30B-A3B attention.
        {"name": "attn_chunk2k_16k_fp8", "kind": "attn", "b": 1, "new": 2048, "len": 16384, "ragged": False, "hq": 32,
         "hkv": 4, "d": 128, "io": "bf16", "kv": "fp8", "window": 0, "sinks": 0, "col": False},
        # A chunk through a sliding window in the activations' column-major
        # layout and in fp32, TinyLlama attention.
        {"name": "attn_chunk1000_f32", "kind": "attn", "b": 1, "new": 1000, "len": 3001, "ragged": False, "hq": 32,
         "hkv": 4, "d": 64, "io": "f32", "kv": "f16", "window": 512, "sinks": 4, "col": True},
        # The smallest store: one token each of four sequences, YaRN.
        {"name": "rope_b4_one", "kind": "rope", "b": 4, "new": 1, "len": 5000, "ragged": True, "hq": 32, "hkv": 8,
         "d": 64, "io": "f32", "kv": "f16", "rope": 64, "pairs": "half", "scaling": "yarn", "factor": 4.0,
         "base": 5e5, "norm": False, "col": False},
        # A 2048-token chunk far into a long context, Llama-3-8B.
        {"name": "rope_2k_bf16", "kind": "rope", "b": 1, "new": 2048, "len": 40000, "ragged": False, "hq": 32,
         "hkv": 8, "d": 128, "io": "bf16", "kv": "bf16", "rope": 128, "pairs": "half", "scaling": "llama3",
         "factor": 8.0, "base": 5e5, "norm": False, "col": False},
        # Ragged chunks with qkNorm, half of each head rotated in interleaved
        # pairs, fp32 column-major activations, fp8 pages.
        {"name": "rope_ragged_fp8", "kind": "rope", "b": 6, "new": 203, "len": 1000, "ragged": True, "hq": 32,
         "hkv": 4, "d": 128, "io": "f32", "kv": "fp8", "rope": 64, "pairs": "inter", "scaling": "linear",
         "factor": 2.0, "base": 1e6, "norm": True, "col": True},
        # Three sequences forked: the last, part-filled page of each in every
        # layer of a Llama-3.2-1B-shaped model.
        {"name": "copy_fork3", "kind": "copy", "layers": 16, "hkv": 8, "d": 64, "kv": "bf16", "pages": 96, "pairs": 3},
        # A pool compacted after sequences have ended: 200 pages of each of
        # 32 layers moved, Llama-3-8B.
        {"name": "copy_compact200", "kind": "copy", "layers": 32, "hkv": 8, "d": 128, "kv": "bf16", "pages": 512,
         "pairs": 200},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "rope", "copy"])
    d = rng.choice([64, 128])
    hkv = rng.choice([4, 8])
    if kind == "copy":
        pages = _log(rng, 8, 512)
        return {"kind": kind, "layers": rng.choice([1, 16, 24, 32]), "hkv": hkv, "d": d,
                "kv": rng.choice(["bf16", "f16", "fp8"]), "pages": pages, "pairs": _log(rng, 1, max(1, pages * 2 // 5))}
    hq = 32 if hkv == 8 else rng.choice([4, 20, 28, 32])
    io = rng.choice(["bf16", "bf16", "f16", "f32"])
    kv = rng.choice(["f16", "bf16", "fp8"])
    col = rng.random() < 0.25
    if kind == "rope":
        b = rng.choice([1, 2, 5, 16, 32])
        new = 1 if rng.random() < 0.3 else _log(rng, 2, 2048 // b)
        rope = rng.choice([d, d, d // 2])
        return {"kind": kind, "b": b, "new": new, "len": new + _log(rng, 1, 40000 // b), "ragged": b > 1, "hq": hq,
                "hkv": hkv, "d": d, "io": io, "kv": kv, "rope": rope, "pairs": rng.choice(["half", "inter"]),
                "scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "factor": float(rng.choice([2, 4, 8])),
                "base": rng.choice([1e4, 5e5, 1e6]), "norm": rng.random() < 0.5, "col": col}
    shape = rng.choice(["one", "few", "chunk", "mixed"])
    b = {"one": rng.choice([1, 2, 7, 16, 32]), "few": rng.choice([1, 4, 8]), "chunk": rng.choice([1, 1, 2, 4]),
         "mixed": rng.choice([9, 17, 26])}[shape]
    new = {"one": 1, "few": _log(rng, 2, 16), "chunk": _log(rng, 17, 2048 // b), "mixed": _log(rng, 17, 351)}[shape]
    past = _log(rng, 1, {"one": 65536 // max(b, 2), "mixed": 2048}.get(shape, 8192))
    window = 0 if rng.random() < 0.5 else _log(rng, 64, 4096)
    return {"kind": kind, "b": b, "new": new, "len": new + past, "ragged": b > 1, "hq": hq, "hkv": hkv, "d": d,
            "io": io, "kv": kv, "window": window, "sinks": rng.choice([0, 1, 4, 40]) if window else 0, "col": col}


# --- inputs -----------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 23)


def _lens(case):
    """Each sequence's new tokens and its length with them, as the case says."""
    b, new, top = case["b"], case["new"], case["len"]
    if not case["ragged"]:
        return [new] * b, [top] * b
    # Chunks of a large batch differ as they do in continuous batching: every
    # eighth sequence brings a chunk, the others one token each.
    if b > 8 and new > 1:
        news = [max(1, new - 36 * (i // 8)) if i % 8 == 0 else 1 for i in range(b)]
    else:
        news = [max(1, new - new * i // (2 * b)) if i else new for i in range(b)]
    lens = [max(n, top - (top * 5 * i) // (8 * b)) for i, n in enumerate(news)]
    return news, lens


def _acts(g, rows, n, dtype, col):
    """Activations of n tokens: unit normal, one channel in 64 three times as
    large; column-major [rows, n] or token-major [n, rows], rows a little
    apart in memory as a fused projection's outputs are."""
    x = torch.randn(n, rows, device="cuda", generator=g)
    x[:, torch.rand(rows, device="cuda", generator=g) < 1 / 64] *= 3.0
    x = x.to(dtype)
    wide, high = (n, rows) if col else (rows, n)
    buf = torch.empty(high, wide + 64, dtype=dtype, device="cuda")
    view = buf[:, :wide]
    view.copy_(x.t() if col else x)
    return view


def _pages(g, case, lens):
    """K and V pools with a table of shuffled pages, what the cache holds."""
    hkv, d, kv = case["hkv"], case["d"], DTYPES[case["kv"]]
    need = [-(-n // PAGE) for n in lens]
    n_pages = sum(need) + 7
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    pools = [torch.randn(n_pages, hkv, d, PAGE, device="cuda", generator=g).to(kv) for _ in range(2)]
    return pools[0], pools[1], table


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    if case["kind"] == "copy":
        n, pairs = case["pages"], case["pairs"]
        shape = (2 * case["layers"], n, case["hkv"], case["d"], PAGE)
        s["pools"] = torch.empty(shape, dtype=DTYPES[case["kv"]], device="cuda")
        for p in s["pools"]:
            p.copy_(torch.randn(shape[1:], device="cuda", generator=g, dtype=torch.float16).to(p.dtype))
        order = torch.randperm(n, device="cuda", generator=g)[:2 * pairs]
        s["src"], s["dst"] = order[:pairs].contiguous(), order[pairs:].contiguous()
        s["moves"] = torch.stack([s["src"], s["dst"]], 1).to(torch.int32).cpu().contiguous()  # the server's own list
        if own:
            from hippo_leap_amd import attention as A
            s["args"] = A.kv_pages_args(list(s["pools"]))
        return s
    news, lens = _lens(case)
    starts = np.concatenate([[0], np.cumsum(news)])
    n = int(starts[-1])
    io, col, d = DTYPES[case["io"]], case["col"], case["d"]
    s.update(n=n, max_new=max(news), max_len=max(lens), q_start=_int(starts.tolist()), kv_lens=_int(lens))
    s["k"], s["v"], s["table"] = _pages(g, case, lens)
    s["q"] = _acts(g, case["hq"] * d, n, io, col)
    s["out"] = torch.zeros_like(s["q"], memory_format=torch.contiguous_format)
    if case["kind"] == "rope":
        s["k_new"], s["v_new"] = (_acts(g, case["hkv"] * d, n, io, col) for _ in range(2))
        s["wq"], s["wk"] = (0.5 + torch.rand(d, device="cuda", generator=g) for _ in range(2)) if case["norm"] else (None, None)
    if own:
        from hippo_leap_amd import attention as A
        s["batch"] = A.chunk_batch(s["k"], s["v"], s["table"], s["q_start"], s["kv_lens"], n, s["max_new"],
                                   s["max_len"], case["hkv"], d)
        layout = A.HL_ACT_COLMAJOR if col else A.HL_ACT_TOKENMAJOR
        if case["kind"] == "attn":
            s["args"] = A.attn_chunk_args(s["batch"], s["q"], s["out"], case["hq"], act_layout=layout,
                                          window=case["window"], n_sink=case["sinks"])
            s["ws"] = A.attn_chunk_workspace(s["args"])
        else:
            kind = {"none": A.HL_ROPE_SCALE_NONE, "linear": A.HL_ROPE_SCALE_LINEAR,
                    "llama3": A.HL_ROPE_SCALE_LLAMA3, "yarn": A.HL_ROPE_SCALE_YARN}[case["scaling"]]
            style = A.HL_ROPE_HALF_SPLIT if case["pairs"] == "half" else A.HL_ROPE_INTERLEAVED
            s["args"] = A.rope_store_chunk_args(
                s["batch"], s["q"], s["k_new"], s["v_new"], s["out"], case["hq"], case["base"], rope_dim=case["rope"],
                rope_style=style, scaling=A.rope_scaling(kind, case["factor"], original_len=8192.0),
                q_norm_w=s["wq"], k_norm_w=s["wk"], eps=EPS, act_layout=layout)
    return s


# --- the plain forms --------------------------------------------------------
def _tokens(x, col):
    """[n, rows] in 32 bits."""
    return (x.t() if col else x).float()


def _places(s):
    """For each new token: its sequence, its place in the chunk, its position."""
    flat = torch.arange(s["n"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["q_start"], flat, right=True) - 1
    at = flat - s["q_start"][seq]
    count = s["q_start"][1:] - s["q_start"][:-1]
    return seq, at.long(), (s["kv_lens"] - count)[seq].long() + at


def _bits(pool):
    """The pool as whole numbers, which torch can index in every type."""
    return pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)


def _gathered(pool, table):
    """The pages that a table names, [b, hkv, d, length] in 32 bits."""
    p = _bits(pool)[table.long()].view(pool.dtype).float()
    return p.permute(0, 2, 3, 1, 4).reshape(table.shape[0], pool.shape[1], pool.shape[2], -1)


def _attn_plain(s):
    case = s["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    grp, b, t = hq // hkv, case["b"], s["max_new"]
    seq, at, pos = _places(s)
    length = s["table"].shape[1] * PAGE
    k, v = _gathered(s["k"], s["table"]), _gathered(s["v"], s["table"])
    q = torch.zeros(b, t, hq * d, device="cuda")
    q[seq, at] = _tokens(s["q"], case["col"]) * (1.0 / math.sqrt(d))
    where = torch.full((b, t), -1, dtype=torch.int64, device="cuda")
    where[seq, at] = pos
    q = q.reshape(b, t, hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, grp * t, d)
    key = torch.arange(length, device="cuda")
    seen = key <= where[..., None]  # [b, t, length]
    if case["window"]:
        seen &= (where[..., None] - key < case["window"]) | (key < case["sinks"])
    scores = torch.matmul(q, k.contiguous()).reshape(b, hkv, grp, t, length)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(b, hkv, grp * t, length), v.transpose(2, 3).contiguous()).reshape(b, hkv, grp, t, d)
    o = (o / total.clamp_min(1e-30)).permute(0, 3, 1, 2, 4).reshape(b, t, hq * d)[seq, at]
    s["out"].copy_(o.t() if case["col"] else o)
    return s["out"]


def _freqs(case):
    """The rotation of each pair per position, in 64 bits, and the factor of
    cos and sin."""
    r, factor, original = case["rope"], case["factor"], 8192.0
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    f = torch.exp(i * (-2.0 / r) * math.log(case["base"]))
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "llama3":
        turns = original * f / (2 * math.pi)  # over the original context
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 1.0
    if case["scaling"] == "yarn":
        dim = [r * math.log(original / (2 * math.pi * turns)) / (2 * math.log(case["base"])) for turns in (32.0, 1.0)]
        lo, hi = max(0, math.floor(dim[0])), min(r - 1, math.ceil(dim[1]))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def _rope_plain(s):
    case = s["case"]
    hq, hkv, d, r = case["hq"], case["hkv"], case["d"], case["rope"]
    seq, at, pos = _places(s)
    f, gain = _freqs(case)
    angle = pos.double()[:, None] * f
    cos, sin = ((fn(angle) * gain).float()[:, None] for fn in (torch.cos, torch.sin))

    def rotated(x, heads, w):
        x = _tokens(x, case["col"]).reshape(s["n"], heads, d)
        if w is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        rest = x[..., r:]
        if case["pairs"] == "half":
            a, c = x[..., :r // 2], x[..., r // 2:r]
            y = torch.cat([a * cos - c * sin, a * sin + c * cos], -1)
        else:
            a, c = x[..., 0:r:2], x[..., 1:r:2]
            y = torch.stack([a * cos - c * sin, a * sin + c * cos], -1).reshape(s["n"], heads, r)
        return torch.cat([y, rest], -1)

    q = rotated(s["q"], hq, s["wq"]).reshape(s["n"], hq * d)
    s["out"].copy_(q.t() if case["col"] else q)
    k = rotated(s["k_new"], hkv, s["wk"])
    v = _tokens(s["v_new"], case["col"]).reshape(s["n"], hkv, d)
    page, slot = s["table"][seq, pos // PAGE].long(), pos % PAGE
    for pool, x in ((s["k"], k), (s["v"], v)):
        x = x.clamp(-448, 448) if case["kv"] == "fp8" else x  # fp8 caches saturate
        _bits(pool)[page, :, :, slot] = _bits(x.to(pool.dtype))
    return {"q": s["out"], "k": s["k"], "v": s["v"]}


def _copy_plain(s):
    p = _bits(s["pools"])
    p[:, s["dst"]] = p[:, s["src"]]
    return s["pools"]


def run(s):
    kind = s["case"]["kind"]
    if own:
        from hippo_leap_amd import attention as A
        if kind == "attn":
            A.attn_chunk(s["args"], s["ws"])
            return s["out"]
        if kind == "rope":
            A.rope_store_chunk(s["args"])
            return {"q": s["out"], "k": s["k"], "v": s["v"]}
        A.kv_pages_copy(s["args"], s["moves"])
        return s["pools"]
    return {"attn": _attn_plain, "rope": _rope_plain, "copy": _copy_plain}[kind](s)


# --- what cannot be left out ------------------------------------------------
def _visible(case, first, last):
    """Keys seen by positions first .. last - 1 (pairs), and keys read at all."""
    pos = np.arange(first, last, dtype=np.int64)
    w, k = case["window"], case["sinks"]
    if not w:
        return int((pos + 1).sum()), last
    sinks = np.minimum(k, np.maximum(0, pos + 1 - w))
    read = last - max(0, first - w + 1)
    return int((np.minimum(pos + 1, w) + sinks).sum()), read + min(k, max(0, first - w + 1))


def work(case):
    if case["kind"] == "copy":
        page = case["hkv"] * case["d"] * PAGE * BYTES[case["kv"]]
        return {"bytes": 2 * page * case["pairs"] * 2 * case["layers"], "flops": 0}
    news, lens = _lens(case)
    n, io, kv = sum(news), BYTES[case["io"]], BYTES[case["kv"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "rope":
        return {"bytes": n * d * ((2 * hq + 2 * hkv) * io + 2 * hkv * kv), "flops": n * d * (hq + hkv) * 4}
    pairs = keys = 0
    for t, length in zip(news, lens):
        p, k = _visible(case, length - t, length)
        pairs, keys = pairs + p, keys + k
    return {"bytes": keys * hkv * d * 2 * kv + 2 * n * hq * d * io, "flops": 4 * pairs * hq * d}


# --- the definition in 64 bits ----------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "copy":
        n = s["pools"].shape[1]
        come_from = torch.arange(n, device="cuda")
        come_from[s["dst"]] = s["src"]
        return _bits(s["pools"])[:, come_from].view(s["pools"].dtype)  # a copy's values are its inputs'
    news, lens = _lens(case)
    hq, hkv, d, col = case["hq"], case["hkv"], case["d"], case["col"]
    table = s["table"].cpu().numpy()
    if case["kind"] == "attn":
        x = (s["q"].t() if col else s["q"]).double()
        out = torch.empty(s["n"], hq * d, dtype=torch.float64, device="cuda")
        first = 0
        for b, (t, length) in enumerate(zip(news, lens)):
            pages = torch.tensor(table[b, :-(-length // PAGE)].astype(np.int64), device="cuda")
            i = torch.arange(length - t, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            hidden = j > i
            if case["window"]:
                hidden |= (j <= i - case["window"]) & (j >= case["sinks"])
            for h in range(hkv):
                ks, vs = (_bits(p)[:, h][pages].view(p.dtype).double().transpose(0, 1).reshape(d, -1)[:, :length]
                          for p in (s["k"], s["v"]))
                for e in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    z = x[first:first + t, e * d:(e + 1) * d] @ ks.contiguous() / d ** 0.5
                    z[hidden] = -float("inf")
                    out[first:first + t, e * d:(e + 1) * d] = torch.softmax(z, -1) @ vs.t().contiguous()
            first += t
        return out.t().contiguous() if col else out
    r, half = case["rope"], case["rope"] // 2
    freq = [case["base"] ** (-2.0 * i / r) for i in range(half)]
    gain = 1.0
    if case["scaling"] == "linear":
        freq = [f / case["factor"] for f in freq]
    elif case["scaling"] == "llama3":
        out = []
        for f in freq:
            wave = 2 * math.pi / f
            if wave < 8192.0 / 4.0:
                out.append(f)
            elif wave > 8192.0:
                out.append(f / case["factor"])
            else:
                u = (8192.0 / wave - 1.0) / 3.0
                out.append((1 - u) * f / case["factor"] + u * f)
        freq = out
    elif case["scaling"] == "yarn":
        where = lambda turns: r * math.log(8192.0 / (turns * 2 * math.pi)) / (2 * math.log(case["base"]))  # noqa: E731
        lo, hi = max(0, math.floor(where(32.0))), min(r - 1, math.ceil(where(1.0)))
        hi = hi if hi != lo else lo + 0.001
        part = [min(1.0, max(0.0, (i - lo) / (hi - lo))) for i in range(half)]
        freq = [f / case["factor"] * p + f * (1 - p) for f, p in zip(freq, part)]
        gain = 0.1 * math.log(case["factor"]) + 1.0
    pos = np.concatenate([np.arange(length - t, length) for t, length in zip(news, lens)])
    turn = torch.polar(torch.full((len(pos), half), gain, dtype=torch.float64),
                       torch.from_numpy(pos[:, None] * np.asarray(freq)[None])).cuda()

    def spun(x, heads, w):
        x = (x.t() if col else x).double().reshape(len(pos), heads, d).clone()
        if w is not None:
            x = x / (x.square().sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        at = (slice(0, half), slice(half, r)) if case["pairs"] == "half" else (slice(0, r, 2), slice(1, r, 2))
        z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn[:, None]
        x[..., at[0]], x[..., at[1]] = z.real, z.imag
        return x

    q = spun(s["q"], hq, s["wq"]).reshape(len(pos), hq * d)
    pools = []
    seqs = np.repeat(np.arange(len(news)), news)
    page = torch.from_numpy(table[seqs, pos // PAGE].astype(np.int64)).cuda()
    slot = torch.from_numpy(pos % PAGE).cuda()
    for pool, x in ((s["k"], spun(s["k_new"], hkv, s["wk"])),
                    (s["v"], (s["v_new"].t() if col else s["v_new"]).double().reshape(len(pos), hkv, d))):
        p = pool.double()
        p[page, :, :, slot] = x.clamp(-448, 448) if case["kv"] == "fp8" else x
        pools.append(p)
    return {"q": q.t().contiguous() if col else q, "k": pools[0], "v": pools[1]}
