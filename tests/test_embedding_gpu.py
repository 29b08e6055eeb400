"""Embedding lookup and its sorted gradient against their definitions in 64 bits."""
import pytest
import torch

import operator_oracles as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ops():
    from revpp import ops

    ops.check_status()
    return ops


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("n,vocab,width", [(1, 1, 1), (1, 7, 128), (3, 5, 13), (33, 100, 64), (200, 1000, 1024),
                                           (77, 300, 515), (1000, 50, 8), (5, 9, 2050)])
@pytest.mark.parametrize("table", TYPES)
@pytest.mark.parametrize("out", TYPES)
def test_lookup(n, vocab, width, table, out):
    ops, g = _ops(), _gen(n)
    w = torch.randn(vocab, width, device="cuda", generator=g).to(table)
    ids = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    y = torch.full((n, width), float("nan"), device="cuda", dtype=out)
    assert ops.embedding_fwd(ids, w, y, scale=3.7) is y
    want = oracle.embed(ids, w, torch.tensor(3.7, dtype=torch.float32).double().item())
    oracle.within(y, want, oracle.embed_bound(want, out))
    assert ops.check_status() == 0


def test_lookup_strides_shapes_and_types_of_ids():
    ops, g = _ops(), _gen()
    big = torch.randn(40, 96, device="cuda", generator=g)
    for w in (big[:, :64], big[:, 3:67], big[::2, 1:33]):  # wider rows, odd offsets
        H = w.shape[1]
        ids = torch.randint(0, w.shape[0], (4, 5), device="cuda", generator=g)
        for i in (ids, ids.int(), ids.t().contiguous().t()):
            y = torch.zeros(4, 5, H + 6, device="cuda").view(20, H + 6)[:, 2:2 + H]
            ops.embedding_fwd(i, w, y)
            assert torch.equal(y, w[ids.reshape(-1)])
    y = torch.empty(4, 5, 96, device="cuda")
    ids = torch.randint(0, 40, (4, 5), device="cuda", generator=g)
    ops.embedding_fwd(ids, big, y)
    assert torch.equal(y, big[ids])
    ops.embedding_fwd(ids[:0], big, y[:0])


def test_ids_outside_the_table_set_the_status_and_give_zeros():
    ops = _ops()
    w = torch.ones(4, 64, device="cuda")
    ids = torch.tensor([0, -1, 4, 3, 2 ** 40, -2 ** 40], device="cuda")
    y = torch.full((6, 64), 5.0, device="cuda")
    ops.embedding_fwd(ids, w, y)
    torch.cuda.synchronize()
    assert ops.check_status() == 4
    assert torch.equal(y[:, 0].cpu(), torch.tensor([1.0, 0, 0, 1, 0, 0]))
    dw = torch.full((4, 64), 7.0, device="cuda")
    ops.embedding_bwd(torch.ones(6, 64, device="cuda"), ids, dw, accumulate=False)
    torch.cuda.synchronize()
    assert ops.check_status() == 4
    assert torch.equal(dw[:, 0].cpu(), torch.tensor([1.0, 0, 0, 1]))


def _tokens(kind, n, vocab, g):
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), device="cuda", generator=g)
    if kind == "one":  # one run through every chunk
        return torch.full((n,), vocab - 1, device="cuda")
    if kind == "skewed":
        u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)
        return (torch.exp(u * torch.tensor(float(vocab), dtype=torch.float64).log().item()).long() - 1).clamp_(0, vocab - 1)
    raise AssertionError(kind)


@pytest.mark.parametrize("kind,n,vocab,width", [
    ("uniform", 1, 1, 1), ("uniform", 1, 3, 64), ("uniform", 31, 5, 40), ("uniform", 32, 2, 128), ("uniform", 33, 40, 13),
    ("skewed", 1000, 300, 128), ("skewed", 4097, 30522, 64), ("skewed", 9999, 257, 515), ("uniform", 700, 131072, 16),
    ("one", 33, 4, 32), ("one", 64, 1, 24), ("one", 1024, 3, 16), ("one", 1025, 3, 16), ("one", 9001, 200, 72),
    ("skewed", 40000, 2, 256), ("uniform", 5000, 149, 1032), ("skewed", 300001, 500, 8), ("one", 140000, 9, 8),
    ("skewed", 3000, 40000, 24), ("skewed", 140001, 40000, 8), ("uniform", 3000, 131072, 8), ("skewed", 70000, 70000, 8), ("uniform", 900, 140000, 8),
    ("one", 256, 3, 130), ("skewed", 255, 40, 1024), ("skewed", 257, 40, 64), ("uniform", 200, 700, 67), ("skewed", 256, 90, 6)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient(kind, n, vocab, width, dtype, accumulate):
    ops, g = _ops(), _gen(n + vocab)
    ids = _tokens(kind, n, vocab, g)
    dy = torch.randn(n, width, device="cuda", generator=g).to(dtype)
    before = torch.randn(vocab, width, device="cuda", generator=g)
    dw = before.clone() if accumulate else torch.full_like(before, float("nan"))
    ops.embedding_bwd(dy, ids, dw, scale=0.75, accumulate=accumulate)
    want, bound = oracle.embed_grad(dy, ids, vocab, 0.75)
    if accumulate:
        want = want + before.double()
        bound = bound + want.abs() * oracle.U
        untouched = torch.ones(vocab, dtype=torch.bool, device="cuda")
        untouched[ids] = False
        assert torch.equal(dw[untouched], before[untouched])
    oracle.within(dw, want, bound + oracle.tiny(torch.float32))
    again = before.clone() if accumulate else torch.full_like(before, float("inf"))
    ops.embedding_bwd(dy, ids, again, scale=0.75, accumulate=accumulate)
    assert torch.equal(dw, again)  # the same bits
    assert ops.check_status() == 0


@pytest.mark.parametrize("padding", [0, 7, -1])
def test_padding_tokens_add_nothing(padding):
    ops, g = _ops(), _gen(5)
    vocab, n = 50, 600
    ids = torch.randint(0, vocab, (3, n // 3), device="cuda", generator=g)
    ids[torch.rand(3, n // 3, device="cuda", generator=g) < 0.4] = padding % vocab
    dy = torch.randn(3, n // 3, 96, device="cuda", generator=g)
    dw = torch.full((vocab, 96), float("nan"), device="cuda")
    ops.embedding_bwd(dy, ids.int(), dw, padding_idx=padding, accumulate=False)
    want, bound = oracle.embed_grad(dy, ids, vocab, 1.0, padding % vocab)
    oracle.within(dw, want, bound)
    assert not dw[padding % vocab].any()
    ops.embedding_bwd(dy, torch.full_like(ids, padding % vocab), dw, padding_idx=padding, accumulate=False)
    assert not dw.any()
    ops.embedding_bwd(dy[:0], ids[:0], dw.fill_(3.0), accumulate=False)
    assert not dw.any()
    ops.embedding_bwd(dy[:0], ids[:0], dw.fill_(3.0))
    assert (dw == 3).all()


def test_gradient_strides():
    ops, g = _ops(), _gen(6)
    ids = torch.randint(0, 20, (100,), device="cuda", generator=g)
    big = torch.randn(200, 80, device="cuda", generator=g)
    for dy in (big[::2, :64], big[:100, 5:69], big[:100].to(torch.bfloat16)[:, 2:66], big[:1, :64].expand(100, 64)):
        store = torch.full((20, 71), 9.0, device="cuda")
        for off in (0, 1, 4):
            dw = store[:, off:off + 64]
            store.fill_(9.0)
            ops.embedding_bwd(dy, ids, dw, accumulate=False)
            want, bound = oracle.embed_grad(dy, ids, 20, 1.0)
            oracle.within(dw, want, bound)
            outside = torch.ones(71, dtype=torch.bool)
            outside[off:off + 64] = False
            assert (store[:, outside] == 9).all()  # beside the rows


def test_gradient_is_the_difference_of_lookups():
    """The lookup is linear in the table: (f(W + h D) - f(W - h D)) / 2h in the direction D is <dW, D>."""
    ops, g = _ops(), _gen(7)
    vocab, width, n, h = 30, 64, 500, 0.5
    ids = _tokens("skewed", n, vocab, g)
    w, d = (torch.randn(vocab, width, device="cuda", generator=g) for _ in range(2))
    dy = torch.randn(n, width, device="cuda", generator=g)
    up, down = torch.empty_like(dy), torch.empty_like(dy)
    ops.embedding_fwd(ids, w + h * d, up, scale=2.0)
    ops.embedding_fwd(ids, w - h * d, down, scale=2.0)
    quotient = ((up.double() - down.double()) / (2 * h) * dy.double()).sum().item()
    dw = torch.zeros(vocab, width, device="cuda")
    ops.embedding_bwd(dy, ids, dw, scale=2.0)
    _, bound = oracle.embed_grad(dy, ids, vocab, 2.0)
    # up and down: the table's sum and the product round (2 U each); dW within its own bound
    slack = (2 * oracle.U * (up.abs() + down.abs()).double() / (2 * h) * dy.abs().double()).sum() + (bound * d.abs().double()).sum()
    assert abs(quotient - (dw.double() * d.double()).sum().item()) <= slack.item()


def test_streams_and_graphs():
    """Two graphs captured on their own streams replay at the same time with workspaces of their own."""
    ops, g = _ops(), _gen(8)
    ops.embedding_bwd(torch.ones(1, 8, device="cuda"), torch.zeros(1, device="cuda", dtype=torch.long),
                      torch.zeros(1, 8, device="cuda"))  # first use outside of a capture
    runs = []
    for k in range(2):
        vocab, width, n = 100 + 30 * k, 64, 3000
        ids = _tokens("skewed", n, vocab, g)
        w = torch.randn(vocab, width, device="cuda", generator=g)
        dy = torch.randn(n, width, device="cuda", generator=g)
        y, dw = torch.zeros_like(dy), torch.zeros(vocab, width, device="cuda")
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ops.embedding_fwd(ids, w, y)
            ops.embedding_bwd(dy, ids, dw, accumulate=False)
        runs.append((graph, stream, ids, w, dy, y, dw))
    for graph, stream, ids, w, dy, y, dw in runs:  # new inputs in the captured tensors
        ids.copy_(ids.flip(0))
        dy.neg_()
        y.zero_()
        dw.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for graph, stream, ids, w, dy, y, dw in runs:
        assert torch.equal(y, w[ids])
        want, bound = oracle.embed_grad(dy, ids, w.shape[0], 1.0)
        oracle.within(dw, want, bound)


def test_rows_beyond_32_bits():
    """Rows whose offset in elements passes 2^31 (a 16-bit table of 4.3 GB)."""
    ops = _ops()
    vocab, width = 70000, 32768
    w = torch.empty(vocab, width, device="cuda", dtype=torch.bfloat16)
    ids = torch.tensor([65535, 65536, 65537, 69999, 1], device="cuda")
    w[ids] = torch.arange(1, 6, device="cuda", dtype=torch.bfloat16)[:, None]
    y = torch.empty(5, width, device="cuda", dtype=torch.bfloat16)
    ops.embedding_fwd(ids, w, y)
    assert torch.equal(y, w[ids])
    del w
    dw = torch.zeros(vocab, width, device="cuda")
    ops.embedding_bwd(y, ids, dw)
    assert torch.equal(dw[ids], y.float())
    assert torch.count_nonzero(dw[:, 0]).item() == 5
