"""GPU: hl_kv_pages_copy, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pools(n_pools, n_pages, page, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, 256, (n_pages, page), dtype=torch.uint8, device="cuda", generator=g) for _ in range(n_pools)]


def _moves(n_pages, n, seed):
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed))[:2 * n]
    return order.reshape(n, 2).to(torch.int32).contiguous()


def _expect(pools, moves):
    want = [p.clone() for p in pools]
    for w in want:
        w[moves[:, 1].long().cuda()] = w[moves[:, 0].long().cuda()]
    return want


@pytest.mark.parametrize("n_pools,n_pages,page,n", [
    (1, 2, 16, 1), (2, 10, 4096, 5), (3, 50, 16 * 1023, 20), (2, 40, 65536, 20), (2, 700, 2048, 300), (70, 12, 1040, 6),
    (130, 1200, 4096, 520), (1, 6, 1 << 20, 3), (2, 5, 32768, 0)])
def test_copies(hl, n_pools, n_pages, page, n):
    from hippo_leap_amd import attention as A
    print(f"pages {n_pools} {n_pages} {page} {n}", flush=True)
    pools = _pools(n_pools, n_pages, page)
    moves = _moves(n_pages, n, n)
    want = _expect(pools, moves)
    A.kv_pages_copy(A.kv_pages_args(pools), moves)
    moves.fill_(-1)  # the list was consumed
    torch.cuda.synchronize()
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_one_page_to_many(hl):
    from hippo_leap_amd import attention as A
    pools = _pools(4, 9, 4096)
    moves = torch.tensor([[3, i] for i in (0, 1, 8, 5)], dtype=torch.int32)
    want = _expect(pools, moves)
    A.kv_pages_copy(A.kv_pages_args(pools), moves)
    assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_far_pages(hl):
    """Pages past 2^32 bytes of a pool."""
    from hippo_leap_amd import attention as A
    page, n = 65536, 70000
    pool = torch.empty(n, page, dtype=torch.uint8, device="cuda")
    pool[5].fill_(17)
    pool[n - 1].fill_(99)
    A.kv_pages_copy(A.kv_pages_args([pool]), torch.tensor([[5, n - 2], [n - 1, 6]], dtype=torch.int32))
    assert (pool[n - 2] == 17).all() and (pool[6] == 99).all()


def test_captured_copies_keep_their_list(hl):
    from hippo_leap_amd import attention as A
    pools = _pools(3, 700, 1024)
    args, moves = A.kv_pages_args(pools), _moves(700, 300, 3)
    kept = moves.clone()
    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        A.kv_pages_copy(args, moves)
    moves.zero_()
    for i in range(3):
        for p, q in zip(pools, _pools(3, 700, 1024, seed=i + 5)):
            p.copy_(q)
        want = _expect(pools, kept)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, w) for p, w in zip(pools, want))


def test_refused_copy_changes_nothing(hl):
    from hippo_leap_amd import _lib
    from hippo_leap_amd import attention as A
    pools = _pools(2, 10, 256)
    want = [p.clone() for p in pools]
    for bad in ([[0, 1], [1, 2]], [[0, 1], [2, 1]], [[0, 10]], [[4, 4]]):
        with pytest.raises(_lib.HLError):
            A.kv_pages_copy(A.kv_pages_args(pools), torch.tensor(bad, dtype=torch.int32))
    torch.cuda.synchronize()
    assert all(torch.equal(p, w) for p, w in zip(pools, want))
