"""CPU: argument checks of the entry points over paged caches, the frequency
tables and the page bookkeeping.  Nothing here reaches a launch."""
import ctypes
import math
import random

import pytest
import torch

from hippo_leap_amd import _lib
from hippo_leap_amd import attention as A

FAKE = 1 << 20  # aligned, never dereferenced


def _batch(**kw):
    s = _lib.ChunkBatch()
    s.batch, s.n_tokens, s.max_new, s.max_kv = 2, 40, 20, 300
    s.q_start = s.kv_lens = s.block_table = FAKE
    s.n_head_kv, s.head_dim, s.kv_dtype, s.n_pages, s.blocks_per_seq = 4, 64, _lib.HL_F16, 50, 10
    s.k_pages, s.v_pages = 1 << 32, 1 << 33
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _attn(batch=None, **kw):
    a = _lib.AttnChunkArgs()
    a.seqs = _batch(**(batch or {}))
    a.n_head, a.io_dtype, a.act_layout = 8, _lib.HL_BF16, _lib.HL_ACT_TOKENMAJOR
    a.q, a.out = 1 << 34, 1 << 35
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _rope(batch=None, **kw):
    a = _lib.RopeStoreChunkArgs()
    a.seqs = _batch(**(batch or {}))
    a.n_head, a.io_dtype, a.act_layout = 8, _lib.HL_BF16, _lib.HL_ACT_TOKENMAJOR
    a.q, a.k, a.v, a.q_out = 1 << 34, 1 << 35, 1 << 36, 1 << 37
    a.eps = 1e-6
    a.freqs.rope_dim = 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_BATCH = [
    ({"batch": 0}, _lib.HL_EINVAL, "batch"), ({"batch": 65536}, _lib.HL_EINVAL, "batch"),
    ({"head_dim": 96}, _lib.HL_EUNSUPPORTED, "head_dim"), ({"head_dim": 256}, _lib.HL_EUNSUPPORTED, "head_dim"),
    ({"n_head_kv": 3}, _lib.HL_EINVAL, "divisible"), ({"n_head_kv": 0}, _lib.HL_EINVAL, "head counts"),
    ({"kv_dtype": _lib.HL_F32}, _lib.HL_EUNSUPPORTED, "fp16/bf16/fp8"), ({"kv_dtype": 9}, _lib.HL_EINVAL, "kv_dtype"),
    ({"n_tokens": 0}, _lib.HL_EINVAL, "n_tokens"), ({"max_new": 0}, _lib.HL_EINVAL, "max_new"),
    ({"max_new": 41}, _lib.HL_EINVAL, "max_new"), ({"max_kv": 0}, _lib.HL_EINVAL, "max_kv"),
    ({"max_kv": 321}, _lib.HL_ECAPACITY, "blocks_per_seq"),
    ({"max_kv": (1 << 24) + 1, "blocks_per_seq": 1 << 20}, _lib.HL_EUNSUPPORTED, "2^24"),
    ({"blocks_per_seq": 0}, _lib.HL_ECAPACITY, "blocks_per_seq"), ({"n_pages": 0}, _lib.HL_EINVAL, "n_pages"),
    ({"q_start": None}, _lib.HL_EINVAL, "null"), ({"kv_lens": None}, _lib.HL_EINVAL, "null"),
    ({"block_table": None}, _lib.HL_EINVAL, "null"), ({"block_table": FAKE + 2}, _lib.HL_EINVAL, "aligned"),
    ({"n_head_kv": 16385}, _lib.HL_EINVAL, "divisible"),
    ({"k_pages": None}, _lib.HL_EINVAL, "pool"), ({"v_pages": (1 << 33) + 8}, _lib.HL_EINVAL, "16-byte"),
]


@pytest.mark.parametrize("bad", range(len(BAD_BATCH)))
def test_batch_refusals(hl, bad):
    kw, code, text = BAD_BATCH[bad]
    a, r = _attn(kw), _rope(kw)
    assert hl.hl_attn_chunk_workspace_bytes(ctypes.byref(a)) == 0
    assert hl.hl_attn_chunk(ctypes.byref(a), FAKE, 1 << 40, None) == code
    assert text in hl.hl_last_error().decode()
    assert hl.hl_rope_store_chunk(ctypes.byref(r), None) == code
    assert text in hl.hl_last_error().decode()


@pytest.mark.parametrize("kw,text", [
    ({"q": None}, "null q"), ({"out": None}, "null out"), ({"q": (1 << 34) + 1}, "aligned"),
    ({"io_dtype": _lib.HL_FP8}, "io_dtype"), ({"act_layout": 2}, "act_layout"), ({"q_stride": 511}, "stride"),
    ({"out_stride": -1}, "stride"), ({"out_stride": 1 << 41}, "stride"), ({"out": 1 << 34}, "overlaps"),
    ({"out": (1 << 34) + 40 * 512 * 2 - 2}, "overlaps"), ({"out": 1 << 32}, "overlaps"), ({"out": (1 << 33) + 64}, "overlaps"),
    ({"scale": -1.0}, "scale"), ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"), ({"window": -1}, "window"),
    ({"n_sink": -2}, "n_sink"), ({"num_splits": -1}, "num_splits"),
])
def test_attn_refusals(hl, kw, text):
    a = _attn(**kw)
    assert hl.hl_attn_chunk(ctypes.byref(a), FAKE, 1 << 40, None) == _lib.HL_EINVAL
    assert text in hl.hl_last_error().decode()


def test_size_refusals(hl):
    a = _attn({"n_tokens": 1 << 24, "max_new": 1 << 20}, n_head=128, q=1 << 40, out=1 << 44)
    assert hl.hl_attn_chunk(ctypes.byref(a), FAKE, 1 << 40, None) == _lib.HL_EUNSUPPORTED
    a = _attn({"n_head_kv": 1}, n_head=16385, q=1 << 40, out=1 << 44)
    assert hl.hl_attn_chunk(ctypes.byref(a), FAKE, 1 << 40, None) == _lib.HL_EUNSUPPORTED
    a = _attn({"n_tokens": (1 << 24) + 1})
    assert hl.hl_attn_chunk(ctypes.byref(a), FAKE, 1 << 40, None) == _lib.HL_EUNSUPPORTED


def test_attn_workspace(hl):
    a = _attn({"max_kv": 32000, "blocks_per_seq": 1000, "max_new": 1, "n_tokens": 2})
    need = hl.hl_attn_chunk_workspace_bytes(ctypes.byref(a))
    assert need > 65536
    for ws, n, text in ((None, need, "workspace"), (FAKE, need - 1, "needed"), (FAKE + 8, need, "16-byte")):
        assert hl.hl_attn_chunk(ctypes.byref(a), ws, n, None) == _lib.HL_EINVAL
        assert text in hl.hl_last_error().decode()
    a = _attn({"max_kv": 32})
    assert hl.hl_attn_chunk_workspace_bytes(ctypes.byref(a)) == 0
    assert hl.hl_attn_chunk(None, None, 0, None) == _lib.HL_EINVAL


@pytest.mark.parametrize("kw,text", [
    ({"k": None}, "null k"), ({"q_out": None}, "null q_out"), ({"q_out": 1 << 35}, "overlaps k"),
    ({"q_out": (1 << 34) + 2}, "overlaps q"), ({"q_out": 1 << 34, "q_out_stride": 1024}, "overlaps q"),
    ({"v": 1 << 33}, "pages overlap"), ({"q_out": 1 << 32}, "pages overlap"), ({"rope_style": 2}, "rope_style"),
    ({"k_stride": 255}, "stride"), ({"q_norm_w": FAKE + 1}, "aligned"), ({"q_norm_w": FAKE, "eps": -1.0}, "eps"),
    ({"k_norm_w": FAKE, "eps": math.nan}, "eps"),
])
def test_rope_refusals(hl, kw, text):
    a = _rope(**kw)
    assert hl.hl_rope_store_chunk(ctypes.byref(a), None) == _lib.HL_EINVAL
    assert text in hl.hl_last_error().decode()


def test_rope_dim_and_pool_refusals(hl):
    for r in (-2, 3, 66):
        a = _rope()
        a.freqs.rope_dim = r
        assert hl.hl_rope_store_chunk(ctypes.byref(a), None) == _lib.HL_EINVAL
        assert "rope_dim" in hl.hl_last_error().decode()
    a = _rope({"v_pages": (1 << 32) + 64})
    assert hl.hl_rope_store_chunk(ctypes.byref(a), None) == _lib.HL_EINVAL
    assert "pools overlap" in hl.hl_last_error().decode()
    assert hl.hl_rope_store_chunk(None, None) == _lib.HL_EINVAL


def test_freqs_refusals(hl):
    f = _lib.RopeFreqs()
    call = lambda r, b, **kw: hl.hl_rope_freqs_init(  # noqa: E731
        ctypes.byref(f), r, b, ctypes.byref(A.rope_scaling(**kw)) if kw else None)
    for r, b, kw in ((0, 1e4, {}), (3, 1e4, {}), (258, 1e4, {}), (64, 1.0, {}), (64, math.inf, {}), (64, math.nan, {}),
                     (64, 1e4, {"kind": 4}), (64, 1e4, {"kind": -1}), (64, 1e4, {"kind": 1, "factor": 0.5}),
                     (64, 1e4, {"kind": 1, "factor": math.nan}), (64, 1e4, {"kind": 2, "factor": 2.0}),
                     (64, 1e4, {"kind": 2, "factor": 2.0, "original_len": 100.0, "low_freq": 4.0, "high_freq": 4.0}),
                     (64, 1e4, {"kind": 3, "factor": 2.0, "original_len": 100.0, "beta_fast": 1.0, "beta_slow": 2.0}),
                     (64, 1e4, {"kind": 3, "factor": 2.0, "original_len": 100.0, "attn_factor": -1.0})):
        assert call(r, b, **kw) == _lib.HL_EINVAL, (r, b, kw)
    assert hl.hl_rope_freqs_init(None, 64, 1e4, None) == _lib.HL_EINVAL


@pytest.mark.parametrize("base", [1e4, 5e5, 1e6])
@pytest.mark.parametrize("r", [2, 64, 126, 128, 256])
def test_freqs_values(hl, base, r):
    """Both floats together carry the frequency to 2^-45; the ends of the
    scaled bands are those of the formulas."""
    plain = A.rope_freqs(r, base)
    w = [base ** (-2.0 * i / r) / (2 * math.pi) for i in range(r // 2)]
    got = [float(plain.turns_hi[i]) + float(plain.turns_lo[i]) for i in range(r // 2)]
    assert all(abs(g - x) <= 2.0 ** -45 * x for g, x in zip(got, w)) and plain.gain == 1.0
    lin = A.rope_freqs(r, base, A.rope_scaling(_lib.HL_ROPE_SCALE_LINEAR, 4.0))
    assert all(abs(lin.turns_hi[i] - x / 4) <= 2.0 ** -24 * x for i, x in enumerate(w))
    ll = A.rope_freqs(r, base, A.rope_scaling(_lib.HL_ROPE_SCALE_LLAMA3, 8.0, 8192.0))
    yarn = A.rope_freqs(r, base, A.rope_scaling(_lib.HL_ROPE_SCALE_YARN, 8.0, 8192.0))
    assert abs(yarn.gain - (0.1 * math.log(8) + 1)) < 1e-6
    for i, x in enumerate(w):
        turns = 8192.0 * x
        want = x if turns >= 4 else x / 8 if turns <= 1 else x * (turns - 1) / 3 + x / 8 * (4 - turns) / 3
        assert abs(ll.turns_hi[i] - want) <= 2.0 ** -23 * want
        assert x / 8 * (1 - 2e-7) <= yarn.turns_hi[i] <= x * (1 + 2e-7)
        if turns >= 32 * base ** (2.0 / r):
            assert abs(yarn.turns_hi[i] - x) <= 2.0 ** -23 * x
        if turns <= base ** (-2.0 / r):
            assert abs(yarn.turns_hi[i] - x / 8) <= 2.0 ** -23 * x
    assert A.rope_freqs(r, base, A.rope_scaling(_lib.HL_ROPE_SCALE_YARN, 8.0, 8192.0, attn_factor=1.5)).gain == 1.5


def _pages(n_pools=2, n_pages=10, page_bytes=4096, pools=None):
    a = _lib.KvPages()
    a.n_pools, a.n_pages, a.page_bytes = n_pools, n_pages, page_bytes
    a._p = (ctypes.c_void_p * 2)(*(pools or (FAKE, FAKE << 4)))
    a.pools = ctypes.cast(a._p, ctypes.POINTER(ctypes.c_void_p))
    return a


@pytest.mark.parametrize("moves,text", [
    ([(0, 10)], "outside"), ([(-1, 3)], "outside"), ([(10, 3)], "outside"), ([(0, 1), (2, 1)], "written again"),
    ([(0, 1), (1, 2)], "read"), ([(1, 2), (0, 1)], "read"), ([(3, 3)], "read"), ([(0, 1)] * 300, "written again"),
])
def test_copy_refusals(hl, moves, text):
    a = _pages()
    flat = (ctypes.c_int32 * (2 * len(moves)))(*[x for m in moves for x in m])
    assert hl.hl_kv_pages_copy(ctypes.byref(a), flat, len(moves), None) == _lib.HL_EINVAL
    assert text in hl.hl_last_error().decode()


def test_copy_argument_refusals(hl):
    move = (ctypes.c_int32 * 2)(0, 1)
    for a, n in ((_pages(n_pools=0), 1), (_pages(n_pages=0), 1), (_pages(page_bytes=0), 1), (_pages(page_bytes=8), 1),
                 (_pages(pools=(FAKE, None)), 1), (_pages(pools=(FAKE, FAKE + 8)), 1), (_pages(), -1),
                 (_pages(pools=(FAKE, FAKE)), 1), (_pages(pools=(FAKE + 40944, FAKE)), 1)):
        assert hl.hl_kv_pages_copy(ctypes.byref(a), move, n, None) == _lib.HL_EINVAL
    assert hl.hl_kv_pages_copy(ctypes.byref(_pages()), None, 1, None) == _lib.HL_EINVAL
    assert hl.hl_kv_pages_copy(None, move, 1, None) == _lib.HL_EINVAL
    assert hl.hl_kv_pages_copy(ctypes.byref(_pages()), None, 0, None) == _lib.HL_OK
    # pools apart, in descending order: past that check (the move is what is refused)
    bad = (ctypes.c_int32 * 2)(0, 10)
    assert hl.hl_kv_pages_copy(ctypes.byref(_pages(pools=(FAKE + 40960, FAKE))), bad, 1, None) == _lib.HL_EINVAL
    assert "outside" in hl.hl_last_error().decode()


def _table(n):
    return torch.full((n,), -1, dtype=torch.int32)


def test_page_pool_fork_and_copy_on_write(hl):
    pool = A.PagePool(8)
    a, b = _table(4), _table(4)
    assert pool.extend(a, 0, 70) is None and pool.free == 5 and a.tolist() == [0, 1, 2, -1]
    pool.fork(a, b, 70)
    assert b.tolist() == a.tolist() and pool.refs(2) == 2 and pool.free == 5
    assert pool.extend(b, 70, 71) == (2, 3)  # its part-filled page is shared: a copy
    assert b.tolist() == [0, 1, 3, -1] and pool.refs(2) == 1
    assert pool.extend(a, 70, 90) is None    # a's own again
    assert pool.extend(b, 71, 97) is None and b.tolist() == [0, 1, 3, 4]
    pool.release(a)
    assert a.tolist() == [-1] * 4 and pool.free == 4 and pool.refs(0) == 1
    pool.release(b, 1, 2)
    assert b.tolist() == [0, -1, -1, 4] and pool.free == 6
    moves = pool.compact(b.reshape(1, -1))
    assert moves.tolist() == [[4, 1]] and b.tolist() == [0, -1, -1, 1]


def test_page_pool_refusals_change_nothing(hl):
    pool = A.PagePool(3)
    a, b = _table(4), _table(4)
    pool.extend(a, 0, 64)
    state = lambda: (a.tolist(), b.tolist(), pool.free, [pool.refs(i) for i in range(3)])  # noqa: E731
    before = state()
    for code, call in (
            (_lib.HL_ECAPACITY, lambda: pool.extend(a, 64, 128)), (_lib.HL_ECAPACITY, lambda: pool.extend(a, 64, 129)),
            (_lib.HL_EINVAL, lambda: pool.extend(a, 64, 63)), (_lib.HL_EINVAL, lambda: pool.extend(b, 5, 9)),
            (_lib.HL_EINVAL, lambda: pool.fork(a, a, 64)), (_lib.HL_EINVAL, lambda: pool.fork(a, b, 129)),
            (_lib.HL_EINVAL, lambda: pool.release(a, 0, 5)), (_lib.HL_EINVAL, lambda: pool.release(a, -1, 1)),
            (_lib.HL_EINVAL, lambda: pool.release(torch.tensor([0, 2], dtype=torch.int32))),
            (_lib.HL_EINVAL, lambda: pool.release(torch.tensor([0, 0], dtype=torch.int32))),
            (_lib.HL_EINVAL, lambda: pool.release(torch.tensor([1, 7], dtype=torch.int32))),
            (_lib.HL_EINVAL, lambda: pool.compact(torch.tensor([[2]], dtype=torch.int32))),
            (_lib.HL_EINVAL, lambda: pool.refs(3)), (_lib.HL_EINVAL, lambda: A.PagePool(0))):
        with pytest.raises(_lib.HLError) as e:
            call()
        assert e.value.code == code and state() == before
    with pytest.raises(_lib.HLError):
        pool.extend(a.long(), 64, 65)


@pytest.mark.parametrize("seed", range(6))
def test_page_pool_against_a_model(hl, seed):
    """Random extends, forks, releases and compactions, with the contents of
    the pages followed through every copy: each sequence always reads what it
    wrote, and no page leaks."""
    rng = random.Random(seed)
    n_pages, bps = rng.choice([5, 40, 200]), 12
    pool = A.PagePool(n_pages)
    content = [None] * n_pages  # page -> list of 32 values
    seqs = []                   # [table, length, values, first kept block]
    for step in range(400):
        act = rng.random()
        if act < 0.45 or not seqs:
            if not seqs or rng.random() < 0.3:
                seqs.append([_table(bps), 0, [], 0])
            s = rng.choice(seqs)
            new = min(bps * 32, s[1] + rng.randint(1, 50))
            try:
                move = pool.extend(s[0], s[1], new)
            except _lib.HLError as e:
                # no pages left, or forked at a place that a window had left behind
                gone = s[1] % 32 and int(s[0][s[1] // 32]) == -1
                assert e.code == (_lib.HL_EINVAL if gone else _lib.HL_ECAPACITY)
                continue
            if move:
                content[move[1]] = list(content[move[0]])
            for p in range(s[1], new):
                page = int(s[0][p // 32])
                assert pool.refs(page) == 1
                if content[page] is None or p % 32 == 0:
                    content[page] = [None] * 32
                content[page][p % 32] = (step, p)
                s[2].append((step, p))
            s[1] = new
        elif act < 0.65:
            s = rng.choice(seqs)
            t = _table(bps)
            n = rng.randint(0, s[1])
            pool.fork(s[0], t, n)
            seqs.append([t, n, s[2][:n], min(s[3], -(-n // 32))])
        elif act < 0.8:
            s = seqs.pop(rng.randrange(len(seqs)))
            pool.release(s[0])
        elif act < 0.9:
            s = rng.choice(seqs)  # a window leaves whole blocks behind, never the one being filled
            keep = rng.randint(s[3], max(s[3], s[1] // 32))
            pool.release(s[0], s[3], keep - s[3])
            s[3] = keep
        else:
            tables = torch.stack([s[0] for s in seqs])
            for f, t in pool.compact(tables, rng.choice([0, 1, 3, 1000])).tolist():
                assert t < f
                content[t] = content[f]
            for s, row in zip(seqs, tables):
                s[0].copy_(row)
        for s in seqs:
            for p in range(32 * s[3], s[1]):
                assert content[int(s[0][p // 32])][p % 32] == s[2][p]
        held = {}
        for s in seqs:
            for page in s[0].tolist():
                if page >= 0:
                    held[page] = held.get(page, 0) + 1
        assert pool.free == n_pages - len(held)
        assert all(pool.refs(p) == held.get(p, 0) for p in range(n_pages))


def test_wrapper_refusals(hl):
    """What the tensors themselves rule out, before any pointer is taken."""
    k = torch.zeros(4, 2, 64, 32, dtype=torch.float16)
    ok = dict(block_table=torch.zeros(2, 3, dtype=torch.int32), q_start=torch.zeros(3, dtype=torch.int32),
              kv_lens=torch.zeros(2, dtype=torch.int32))
    call = lambda **kw: A.chunk_batch(kw.pop("k", k), kw.pop("v", k), **{**ok, **kw}, n_tokens=4, max_new=2,  # noqa: E731
                                      max_kv=64, n_head_kv=2, head_dim=64)
    for kw in ({"q_start": torch.zeros(3)}, {"kv_lens": torch.zeros(3, dtype=torch.int32)},
               {"block_table": torch.zeros(6, dtype=torch.int32)}, {"k": k[:3]}, {"v": k.to(torch.bfloat16)},
               {"block_table": torch.zeros(3, 2, dtype=torch.int32).t()}, {}):  # the last: not on the GPU
        with pytest.raises(_lib.HLError):
            call(**kw)
    with pytest.raises(_lib.HLError):
        A.kv_pages_copy(_pages(), torch.zeros(1, 2))
    with pytest.raises(_lib.HLError):
        A.kv_pages_args([k, k[:2]])
    x = torch.zeros(1, 128)
    for t in (x.expand(4, 128), torch.zeros(128, 4).t(), torch.zeros(4, 64), torch.zeros(512)):
        with pytest.raises(_lib.HLError):
            A._act(t, 128, 4, _lib.HL_ACT_TOKENMAJOR, "q")


def test_another_device_is_refused(hl, monkeypatch):
    """Arguments made for one device, called with another one current or on
    another one's stream: refused before the library is asked."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    a, r, p = _attn(), _rope(), _pages()
    for args, call in ((a, A.attn_chunk), (r, A.rope_store_chunk),
                       (p, lambda x, **kw: A.kv_pages_copy(x, torch.zeros(1, 2, dtype=torch.int32), **kw))):
        args._device = 1
        with pytest.raises(_lib.HLError) as e:
            call(args)
        assert "cuda:1" in str(e.value)

    class Stream:
        device = torch.device("cuda", 0)
        cuda_stream = 0
    with pytest.raises(_lib.HLError):
        A.attn_chunk(a, stream=Stream())
    with pytest.raises(_lib.HLError):
        A._device_of(torch.zeros(1), torch.zeros(1, device="meta"))
