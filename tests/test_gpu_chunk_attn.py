"""GPU: hl_attn_chunk against the plain implementation in 64 bits."""
import math

import pytest
import torch

from paged_util import PAGE, Case, attn_reference, check_attn

pytestmark = pytest.mark.gpu

# news, lens, hq, hkv, d, io, kv, window, sinks, col
CASES = {
    "first_token": ([1], [1], 4, 4, 64, "f32", "f16", 0, 0, False),
    "one_page": ([1], [32], 8, 2, 64, "bf16", "bf16", 0, 0, False),
    "page_and_one": ([1], [33], 8, 2, 128, "f16", "f16", 0, 0, False),
    "one_long": ([1], [5000], 32, 8, 64, "f32", "f16", 0, 0, False),
    "one_long_bf16_f32": ([1], [3333], 32, 4, 128, "f32", "bf16", 0, 0, False),
    "one_fp8": ([1], [777], 32, 8, 128, "bf16", "fp8", 0, 0, False),
    "one_fp8_f32": ([1], [777], 32, 4, 64, "f32", "fp8", 0, 0, True),
    "batch_decode": ([1] * 7, [1, 31, 32, 33, 700, 65, 1999], 32, 8, 128, "bf16", "bf16", 0, 0, False),
    "window_one": ([1, 1], [90, 200], 8, 8, 64, "f32", "bf16", 1, 0, False),
    "window_sinks": ([1, 3], [1500, 1501], 32, 8, 64, "f32", "f16", 1024, 4, False),
    "window_longer": ([5], [100], 8, 2, 128, "f16", "f16", 5000, 4, False),
    "sinks_past_window": ([4], [300], 8, 2, 64, "bf16", "bf16", 16, 100, False),
    "sinks_past_end": ([2], [50], 8, 2, 64, "bf16", "f16", 3, 1000, False),
    "verify": ([5, 1, 0, 4], [2049, 1, 64, 500], 32, 8, 128, "bf16", "bf16", 0, 0, False),
    "whole_prompt": ([100], [100], 8, 2, 64, "bf16", "bf16", 0, 0, False),
    "whole_prompt_col": ([257], [257], 16, 2, 128, "f16", "f16", 0, 0, True),
    "chunk": ([130], [515], 32, 8, 128, "bf16", "bf16", 0, 0, False),
    "chunk_fp8": ([77], [300], 32, 4, 128, "bf16", "fp8", 0, 0, False),
    "chunk_f32_bf16": ([70], [333], 16, 4, 128, "f32", "bf16", 0, 0, True),
    "chunk_f32_fp8": ([65], [129], 8, 2, 64, "f32", "fp8", 40, 3, False),
    "chunk_f16_on_bf16": ([40], [111], 8, 4, 64, "f16", "bf16", 0, 0, False),
    "chunk_window": ([300], [900], 16, 4, 64, "f32", "f16", 128, 4, True),
    "chunk_window_wide": ([200], [1000], 8, 8, 128, "bf16", "bf16", 333, 40, False),
    "group_5": ([33, 2], [100, 40], 20, 4, 64, "bf16", "bf16", 0, 0, False),
    "group_7": ([19], [219], 28, 4, 128, "bf16", "f16", 50, 1, False),
    "one_kv_head_20": ([3, 1], [80, 999], 20, 1, 128, "f32", "f16", 0, 0, False),
    "one_kv_head_64": ([1, 17], [70, 300], 64, 1, 64, "bf16", "bf16", 0, 0, False),
    "no_groups": ([45, 1], [45, 600], 4, 4, 128, "f16", "f16", 0, 0, True),
    "mixed": ([1, 350, 1, 0, 120, 1, 2], [1000, 700, 33, 0, 120, 2000, 5], 32, 8, 64, "f16", "f16", 0, 0, False),
    "mixed_window": ([1, 64, 1, 300], [4000, 2000, 50, 300], 16, 2, 128, "bf16", "bf16", 500, 5, False),
    "many": ([1, 2, 3] * 50, [40, 2, 77] * 50, 8, 2, 64, "bf16", "bf16", 0, 0, False),
    "big_chunk": ([1500], [2600], 8, 2, 128, "bf16", "bf16", 0, 0, False),
    # windows that nothing leaves, tokens at positions below zero
    "window_endless": ([40, 3, 1], [30, 90, 700], 8, 2, 64, "bf16", "bf16", 2**31 - 1, 2**31 - 1, False),
    "window_endless_tiles": ([300], [200], 8, 2, 128, "f16", "f16", 2**31 - 1, 4, False),
    "window_all_but_one": ([70, 2], [700, 641], 8, 2, 64, "bf16", "fp8", 699, 2**31 - 1, False),
    # enough row blocks for the 8-wave form (head dim 128, 256 blocks of 256 rows)
    "eight_waves": ([2048], [2300], 32, 8, 128, "bf16", "bf16", 0, 0, False),
    "eight_waves_fp8": ([1700, 1, 500], [1700, 900, 2111], 32, 8, 128, "bf16", "fp8", 0, 0, False),
    "eight_waves_f16_window": ([33, 2050, 0, 40], [4000, 2050, 100, 95], 32, 8, 128, "f16", "f16", 700, 40, True),
    "eight_waves_nothing": ([2300], [1900], 32, 8, 128, "bf16", "bf16", 0, 0, False),
}


@pytest.mark.parametrize("name", CASES)
def test_matches_plain(hl, name):
    from hippo_leap_amd import attention as A
    news, lens, hq, hkv, d, io, kv, window, sinks, col = CASES[name]
    print(f"attn {name}", flush=True)
    c = Case(news, lens, hq, hkv, d, io, kv, col, lead=2, tail=3, seed=len(name))
    c.run_attn(A, window, sinks)
    worst = check_attn(c, window=window, n_sink=sinks)
    print(f"  {worst:.3f} of the bound", flush=True)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("new", [1, 6, 70])
def test_any_split(hl, splits, new):
    from hippo_leap_amd import attention as A
    print(f"splits {splits} new {new}", flush=True)
    c = Case([new, 1], [1111, 40], 16, 4, 128, "f32", "bf16", seed=splits)
    for _ in range(2):  # the counters are left as they were found
        c.out.fill_(77)
        c.run_attn(A, num_splits=splits)
        check_attn(c)


@pytest.mark.parametrize("col", [False, True])
@pytest.mark.parametrize("io", ["f32", "f16", "bf16"])
def test_strides_and_alignment(hl, col, io):
    """Rows a little apart, and tensors that begin one element into their
    buffers: any alignment of whole elements is taken."""
    from hippo_leap_amd import attention as A
    print(f"strides {col} {io}", flush=True)
    for pad in (1, 8, 64):
        c = Case([37, 1, 5], [300, 77, 5], 8, 2, 64, io, "f16", col, lead=1, tail=2, pad=pad, seed=pad)
        for name in ("q", "out"):
            t = getattr(c, name)
            buf = torch.full((t.shape[0] * t.stride(0) + 16,), 77.0, dtype=t.dtype, device="cuda")
            moved = torch.as_strided(buf, t.shape, t.stride(), 1 if pad != 8 else 8)
            moved.copy_(t)
            setattr(c, name, moved)
        c.run_attn(A, window=100, n_sink=2)
        check_attn(c, window=100, n_sink=2)


def test_scale_and_large_scores(hl):
    from hippo_leap_amd import attention as A
    for io, kv, gain in (("f32", "f16", 6.0), ("bf16", "bf16", 4.0), ("f32", "bf16", 5.0)):
        print(f"large {io} {kv}", flush=True)
        c = Case([20, 1], [200, 90], 8, 2, 64, io, kv, gain=gain)
        c.run_attn(A, scale=0.05)
        check_attn(c, scale=0.05)


def test_tiny_and_huge_queries(hl):
    """Each row's q has a scale of its own: rows of 2^-100 and of 2^90 beside
    ordinary ones, with fp16 operands."""
    from hippo_leap_amd import attention as A
    c = Case([6], [64], 4, 2, 64, "f32", "f16")
    c.q[0] *= 2.0 ** -100
    c.q[3] *= 2.0 ** -130  # below fp32's normal range
    c.q[4] = 0
    c.run_attn(A)
    check_attn(c)
    c.q[1] *= 2.0 ** 90  # the softmax becomes a choice of the largest score
    c.run_attn(A)
    ref, _ = attn_reference(c)
    assert (c.tokens(c.out) - ref).abs().max() < 1e-5


def test_rows_that_see_nothing(hl):
    """Lengths below the chunk (positions below zero), lengths of zero, and
    pages that are not in the pool: zeros."""
    from hippo_leap_amd import attention as A
    for news, lens in (([5, 3], [2, 0]), ([40], [33]), ([200, 1], [150, 0])):
        print(f"nothing {news} {lens}", flush=True)
        c = Case(news, lens, 8, 2, 64, "bf16", "bf16", tail=1)
        c.run_attn(A)
        check_attn(c)
        for b, (t, n) in enumerate(zip(news, lens)):
            assert (c.tokens(c.out)[c.starts[b]:c.starts[b] + max(0, t - n)] == 0).all()
    for new in (1, 64):
        c = Case([new], [200], 8, 2, 128, "f32", "f16")
        c.table[0, 2] = c.n_pages
        c.table[0, 4] = -1
        c.run_attn(A)
        check_attn(c, hidden_pages=(2, 4))
        c.table[0, :] = -1
        c.run_attn(A)
        assert (c.tokens(c.out) == 0).all()


@pytest.mark.parametrize("new,window", [(1, 64), (1, 100), (7, 50), (90, 130)])
def test_pages_outside_the_window_are_not_needed(hl, new, window):
    """What lies between the sinks and the window may have been given back: its
    table entries, and NaN in the pages of its neighbours, do not matter."""
    from hippo_leap_amd import attention as A
    length = 800
    c = Case([new], [length], 8, 2, 64, "bf16", "bf16", seed=new)
    c.run_attn(A, window, 5)
    check_attn(c, window=window, n_sink=5)
    before = c.out.clone()
    first = (length - new - window + 1) // PAGE
    for t in range(1, first):
        c.k.view(torch.int16)[c.pages[0][t]] = 0x7FC0
        c.v.view(torch.int16)[c.pages[0][t]] = 0x7FC0
        c.table[0, t] = -1 if t % 2 else 2 ** 31 - 1
    c.run_attn(A, window, 5)
    assert torch.equal(c.out, before)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("new,kv,heads,d", [(3, "f16", (8, 2), 64), (50, "bf16", (8, 2), 64), (300, "bf16", (8, 2), 64),
                                            (300, "f16", (8, 2), 64), (2060, "bf16", (32, 8), 128)])
def test_not_finite_reaches_only_who_sees_it(hl, value, which, new, kv, heads, d):
    """An inf or NaN at a new token's k or v, and at one that the window has
    left behind for some rows: the other rows keep their finite results."""
    from hippo_leap_amd import attention as A
    print(f"{which} {value} new {new}", flush=True)
    length, window = new + 70, 60
    c = Case([new], [length], *heads, d, "bf16", kv, seed=new)
    c.run_attn(A, window, 2)
    clean = c.tokens(c.out)
    marks = [length - 2, length - new - window + 2][:1 if new < 4 else 2]  # both would reach each of 3 rows
    for j in marks:
        if j >= 2:
            getattr(c, which)[c.pages[0][j // PAGE], :, 5, j % PAGE] = value
    c.run_attn(A, window, 2)
    got = c.tokens(c.out)
    pos = torch.arange(length - new, length, device="cuda")
    touched = torch.zeros(new, dtype=torch.bool, device="cuda")
    for j in marks:
        if j >= 2:
            touched |= (pos >= j) & (pos - j < window)
    assert touched.any() and not touched.all()
    # whole-tile and key-by-key sums round apart
    assert (got[~touched] - clean[~touched]).abs().max() <= 2 ** -6 * clean.abs().max()
    if which == "v":
        ref, _ = attn_reference(c, window=window, n_sink=2)
        hit = got[touched].reshape(-1, c.hq, c.d)[:, :, 5]
        want = ref[touched].reshape(-1, c.hq, c.d)[:, :, 5]
        assert torch.equal(torch.isnan(hit), torch.isnan(want))
        assert torch.equal(hit[~torch.isnan(hit)], want[~torch.isnan(want)])
        rest = got[touched].reshape(-1, c.hq, c.d)[:, :, 6:]
        assert torch.isfinite(rest).all()
    elif not (value == -math.inf or value == math.inf):
        assert torch.isnan(got[touched]).all()


@pytest.mark.parametrize("new,io,kv", [(1, "f32", "f16"), (40, "bf16", "bf16"), (40, "f32", "fp8")])
def test_contexts_beyond_the_page_table_in_lds(hl, new, io, kv):
    """One workgroup walks more pages (2048 and more) than its table holds;
    pages missing before and after that point."""
    from hippo_leap_amd import attention as A
    print(f"long {new} {io} {kv}", flush=True)
    c = Case([new], [140001], 4, 1, 64, io, kv, seed=new)
    c.table[0, 7] = -1
    c.table[0, 4000] = c.n_pages
    for splits in (1, 2, 0):
        c.out.fill_(77)
        c.run_attn(A, num_splits=splits)
        check_attn(c, hidden_pages=(7, 4000))


@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("d,io,kv", [(64, "bf16", "bf16"), (64, "f32", "f16"), (64, "f16", "fp8"), (128, "bf16", "bf16"),
                                     (128, "f16", "f16"), (128, "f32", "bf16"), (128, "bf16", "fp8")])
def test_single_tokens_beside_chunks(hl, d, io, kv, splits):
    """One token over more than 64 tiles per wave beside chunks, in one launch or two;
    pages missing in both; groups of 16 and of 17 to 32 rows."""
    from hippo_leap_amd import attention as A
    for hq in (8, 32):
        print(f"beside {d} {io} {kv} {splits} {hq}", flush=True)
        c = Case([1, 100, 1, 0, 41, 1], [9001, 700, 8300, 5, 41, 1], hq, 1, d, io, kv, seed=hq)
        c.table[:, 2] = -1
        c.table[0, 270] = c.n_pages
        for _ in range(2):
            c.out.fill_(77)
            c.run_attn(A, num_splits=splits)
            check_attn(c, hidden_pages=(2, 270))


def test_missing_pages_in_the_eight_wave_form(hl):
    from hippo_leap_amd import attention as A
    for kv in ("bf16", "fp8"):
        c = Case([2048], [2200], 32, 8, 128, "bf16", kv)
        c.table[0, 3] = -1
        c.table[0, 66] = c.n_pages + 1
        c.run_attn(A, 1000, 4)
        check_attn(c, window=1000, n_sink=4, hidden_pages=(3, 66))


def test_offsets_past_32_bits(hl):
    """Pages more than 2^32 bytes, and 2^31 elements, into their pools."""
    from hippo_leap_amd import attention as A
    c = Case([2, 60], [100, 90], 8, 8, 128, "bf16", "bf16")
    n = 70000
    far = [torch.empty(n, c.hkv, c.d, PAGE, dtype=c.kv, device="cuda") for _ in range(2)]
    for pool, small in zip(far, (c.k, c.v)):
        pool[n - c.n_pages:] = small
    c.k, c.v = far
    c.table += n - c.n_pages
    c.pages = [[p + n - c.n_pages for p in row] for row in c.pages]
    c.run_attn(A)
    check_attn(c)


def test_replays_with_other_lists(hl):
    """A captured call reads its lists when it runs: lengths, chunks and pages
    change between replays; eager calls of another shape run in between on the
    same workspace."""
    from hippo_leap_amd import attention as A
    c = Case([1, 40, 1], [900, 300, 64], 16, 4, 64, "f32", "f16")
    other = Case([6], [2000], 32, 8, 128, "bf16", "bf16")
    a = A.attn_chunk_args(c.batch(A, max_new=42, max_kv=928), c.q, c.out, c.hq, act_layout=c.layout(A))
    b = A.attn_chunk_args(other.batch(A), other.q, other.out, other.hq, act_layout=other.layout(A))
    big = max((a, b), key=A.attn_chunk_workspace_bytes)
    ws = A.attn_chunk_workspace(big)
    A.attn_chunk(a, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.attn_chunk(a, ws)
    for news, lens in (([1, 40, 1], [900, 300, 64]), ([42, 0, 0], [899, 299, 1]), ([0, 1, 41], [0, 1, 64]),
                       ([14, 14, 14], [450, 290, 50])):
        print(f"replay {news} {lens}", flush=True)
        c.news, c.lens = news, lens
        c.starts = [0, news[0], news[0] + news[1], 42]
        c.q_start.copy_(torch.tensor(c.starts, dtype=torch.int32))
        c.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        c.out.fill_(77)
        other.out.fill_(77)
        A.attn_chunk(b, ws)
        graph.replay()
        A.attn_chunk(b, ws)
        torch.cuda.synchronize()
        check_attn(c)
        check_attn(other)


def test_streams_and_repeats(hl):
    """On a stream of the caller's, with a workspace each, two calls at once;
    repeats are bit-identical."""
    from hippo_leap_amd import attention as A
    cases = [Case([1] * 4, [3000, 2000, 100, 1], 32, 8, 64, "f32", "f16", seed=i) for i in range(2)]
    args = [A.attn_chunk_args(c.batch(A), c.q, c.out, c.hq, act_layout=c.layout(A)) for c in cases]
    spaces = [A.attn_chunk_workspace(a) for a in args]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    first = None
    for _ in range(3):
        for a, ws, st in zip(args, spaces, streams):
            A.attn_chunk(a, ws, stream=st)
        torch.cuda.synchronize()
        for c in cases:
            check_attn(c)
        if first is None:
            first = [c.out.clone() for c in cases]
        assert all(torch.equal(c.out, f) for c, f in zip(cases, first))


def test_lists_outside_the_bounds_stay_inside_the_buffers(hl):
    """Lists that break the host's bounds (chunks past n_tokens, starts that go
    back, lengths past the table): unspecified outputs, nothing else written."""
    from hippo_leap_amd import attention as A
    c = Case([3, 50], [100, 200], 8, 2, 64, "bf16", "bf16", lead=0, tail=0)
    guard = torch.full((c.n + 64, c.hq * c.d), 55.0, dtype=c.io, device="cuda")
    c.out = guard[32:32 + c.n]
    for starts, lens in (([0, 3, 5000], [100, 200]), ([40, 3, 53], [100, 10 ** 9]), ([-5, 60, 20], [-3, 224])):
        print(f"lists {starts} {lens}", flush=True)
        c.q_start.copy_(torch.tensor(starts, dtype=torch.int32))
        c.kv_lens.copy_(torch.tensor(lens, dtype=torch.int32))
        c.run_attn(A, max_kv=c.bps * PAGE)
        torch.cuda.synchronize()
        assert (guard[:32] == 55).all() and (guard[32 + c.n:] == 55).all()
