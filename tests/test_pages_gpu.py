"""Copies of cache pages, bit for bit."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def pages():
    from llm_infer_rust_b200.kernels import pages as m
    return m


def pool(n, heads, page, dim, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n + heads + dim)
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, heads, page, dim), generator=g, dtype=torch.int64).to(torch.int32)     # NaN among them
    return (bits.view(torch.float32) if dtype == F32 else bits.to(torch.int16).view(BF16)).to(DEV)


def same(a, b):
    whole = torch.int32 if a.element_size() == 4 else torch.int16
    return torch.equal(a.view(whole), b.view(whole))


def check(tensors, moves):
    want = [t.clone() for t in tensors]
    for w, t in zip(want, tensors):
        for a, b, n in moves:
            w[b, :, :n] = t[a, :, :n]
    pages().PageCopier(tensors).copy(moves)
    assert all(same(t, w) for t, w in zip(tensors, want))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,page,dim", [(8, 16, 128), (1, 1, 1), (3, 5, 7), (2, 24, 10), (5, 32, 48), (1, 64, 256), (40, 2, 2)])
def test_forks_and_moves(dtype, heads, page, dim):
    tensors = [pool(20, heads, page, dim, dtype, seed=s) for s in range(3)]
    check(tensors, [(4, 9, page), (4, 1, (page + 1) // 2), (19, 0, 1), (3, 2, 0), (7, 18, page - 1)])


def test_tensors_of_unlike_heads_and_types():
    tensors = [pool(9, 4, 16, 128, BF16), pool(9, 1, 16, 576, BF16), pool(9, 2, 16, 64, F32), pool(9, 3, 16, 33, BF16)]
    check(tensors, [(1, 2, 16), (1, 3, 7), (8, 4, 15)])


def test_bases_off_16_bytes():
    flat = pool(1, 1, 1, 9 * 2 * 16 * 64 + 2, BF16).reshape(-1)
    check([flat[1:-1].view(9, 2, 16, 64)], [(1, 2, 16), (1, 3, 7)])


@pytest.mark.parametrize("n", [1, 2, 16, 17, 64, 65, 500, 2048, 2049, 5000])
def test_many_moves(n):
    total = 2 * n + 3
    order = torch.randperm(total, generator=torch.Generator().manual_seed(n)).tolist()
    check([pool(total, 2, 4, 8, BF16), pool(total, 1, 4, 16, F32)], [(order[i], order[n + i], 1 + i % 4) for i in range(n)])


def test_one_page_to_many():
    check([pool(300, 8, 16, 128, BF16) for _ in range(2)], [(5, 10 + i, 11) for i in range(200)])


def test_pages_beyond_2_31_elements():
    t = torch.zeros(70000, 8, 32, 128, dtype=BF16, device=DEV)                  # 4.6 GB, 2.3 G elements
    t[69999] = pool(1, 8, 32, 128, BF16)[0]
    pages().PageCopier([t]).copy([(69999, 69998, 32), (69999, 1, 5)])
    assert same(t[69998], t[69999]) and same(t[1, :, :5].contiguous(), t[69999, :, :5].contiguous()) and not t[1, :, 5:].any()


def test_moves_as_a_tensor_and_none():
    t = pool(9, 2, 4, 8, F32)
    c = pages().PageCopier([t])
    before = t.clone()
    c.copy([])
    c.copy(torch.zeros((0, 3), dtype=torch.int32))
    assert same(t, before)
    moves = torch.tensor([[1, 2, 4], [3, 4, 2]], dtype=torch.int32)
    c.copy(moves)
    moves.zero_()                                                               # (read before the call returned)
    before[2], before[4, :, :2] = before[1], before[3, :, :2]
    assert same(t, before)


def test_streams_and_graphs():
    t = pool(50, 2, 16, 64, BF16)
    c = pages().PageCopier([t])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.copy([(1, 2, 16), (3, 4, 5)])
    t[1].fill_(2.0)
    t[3].fill_(3.0)
    graph.replay()
    torch.cuda.synchronize()
    assert (t[2] == 2.0).all() and (t[4, :, :5] == 3.0).all() and not (t[4, :, 5:] == 3.0).any()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t[10].fill_(5.0)
        c.copy([(10, 11, 16)])
    c.copy([(1, 12, 16)])
    torch.cuda.synchronize()
    assert (t[11] == 5.0).all() and (t[12] == 2.0).all()


@pytest.mark.parametrize("moves", [[(0, 1, 4), (2, 1, 4)], [(0, 1, 4), (1, 2, 4)], [(3, 3, 4)], [(0, 9, 4)], [(-1, 2, 4)], [(0, 2, 5)], [(0, 2, -1)],
                                   [(i, 40 + i, 4) for i in range(20)] + [(3, 45, 1)], [(i, 40 + i, 4) for i in range(20)] + [(41, 80, 1)]])
def test_refused_moves_change_nothing(moves):
    t = pool(9 if max(max(m[:2]) for m in moves) < 10 else 100, 2, 4, 8, F32)
    before = t.clone()
    with pytest.raises(pages().KernelError, match="a move names a page outside|is the target of two moves"):
        pages().PageCopier([t]).copy(moves)
    assert same(t, before)


def test_refused_tensors():
    m = pages()
    t = pool(9, 2, 4, 8, F32)
    for tensors in ([], [t[0]], [t.transpose(1, 2)], [t, pool(8, 2, 4, 8, F32)], [t, pool(9, 2, 5, 8, F32)], [t, t], [t.to(torch.uint8)], [t.double()],
                    [t[:0]], [t, t.cpu()]):
        with pytest.raises(m.KernelError):
            m.PageCopier(tensors)
    c = m.PageCopier([t])
    for moves in (torch.zeros(1, 3, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 3, dtype=torch.int32, device=DEV),
                  torch.zeros(3, dtype=torch.int32), torch.zeros(2, 6, dtype=torch.int32)[:, ::2]):
        with pytest.raises(m.KernelError, match="moves are int32"):
            c.copy(moves)
